"""GPU: norms around a gated residual branch against their definition in 64 bits (forward, gradients by torch's differentiation of
the definition, and by differences), in both layouts, every gate, odd sizes, strides, streams and capture; and the run of
them as used: a stack of the framework's dense blocks trained with the AdamW step."""
import math

import pytest
import torch

from helpers import O as ORACLE, pkg
from optim_ref import step64

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def R():
    return pkg("residual")


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def rows_of(t, dim):
    """[pixels, C] in 64 bits on the CPU."""
    t = t.detach().double().cpu()
    return (t.movedim(1, -1) if dim == 1 else t).reshape(-1, t.shape[dim])


def norm64(z, spec):
    if spec is None:
        return z
    w = spec.weight.detach().double().cpu() if spec.weight is not None else 1.0
    b = spec.bias.detach().double().cpu() if spec.bias is not None else 0.0
    if spec.kind == "none":
        return z * w + b
    if spec.kind == "layer":
        z = z - z.mean(1, keepdim=True)
    return z / torch.sqrt((z * z).mean(1, keepdim=True) + spec.eps) * w + b


def gate64(gate, x, act, dim):
    if gate is None:
        return 1.0
    g = gate.detach().double().cpu()
    if gate.shape == x.shape:
        g = rows_of(gate, dim)
    elif gate.dim() == 2:
        g = g.repeat_interleave(x.numel() // (x.shape[0] * x.shape[dim]), 0)
    return torch.sigmoid(g) if act == "sigmoid" else g


def spec_of(kind, c, weights, gen, dtype=F32):
    if kind is None:
        return None
    rand = lambda s, m: (m + s * torch.randn(c, generator=gen)).to(DEV, dtype)  # noqa: E731
    w = rand(0.2, 1.0) if weights else None
    b = rand(0.2, 0.0) if weights and kind == "layer" or (weights and kind == "none") else None
    return R().NormSpec(kind, w, b, 1e-5)


def make(shape, dim, dtype, post, gate, pre, weights=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    c = shape[dim]
    rand = lambda s=shape: torch.randn(s, generator=g)  # noqa: E731
    per_c = [1] * len(shape)
    per_c[dim] = c
    x = (rand() + 0.5 * rand(per_c)).to(DEV, dtype)
    f = (rand() * (1 + rand(per_c).abs()) + 0.3).to(DEV, dtype)
    q = {None: None, "channel": lambda: (0.5 + 0.3 * rand((c,))).to(DEV), "image": lambda: (0.5 + 0.3 * rand((shape[0], c))).to(DEV),
         "full": lambda: rand().to(DEV, dtype)}[gate]
    return x, f, q() if q else None, spec_of(post, c, weights, g), spec_of(pre, c, weights, g)


def limits(x, f, gate, post, pre, act, scale, dim):
    """Largest magnitudes that enter the results; what follows is derived from them.

    A sum over C channels runs over at most 16 terms a thread and 10 levels of a tree (26 roundings; twice for a
    variance about a mean), a product chain over at most 10 factors: 64 u of the largest term covers each stage's own
    error, and what a stage passes on is multiplied by the next one's slope (r |w|)."""
    big = lambda t: float(t.detach().abs().max()) if torch.is_tensor(t) else abs(t)  # noqa: E731
    lim = {}
    X, Fr = rows_of(x, dim), rows_of(f, dim)

    def unit(z, spec):
        """(n, largest n, largest factor r) before weight and bias"""
        if spec is None or spec.kind == "none":
            return z, big(z), 1.0
        zc = z - z.mean(1, keepdim=True) if spec.kind == "layer" else z
        r = 1 / torch.sqrt((zc * zc).mean(1, keepdim=True) + spec.eps)
        return zc * r, big(zc * r) + (big(z) * float(r.max()) if spec.kind == "layer" else 0.0), float(r.max())
    w2 = big(post.weight) if post is not None and post.weight is not None else 1.0
    b2 = big(post.bias) if post is not None and post.bias is not None else 0.0
    G = gate64(gate, x, act, dim)
    lim["n_f"], lim["nf"], lim["rf"] = unit(Fr, post)
    lim["a"] = lim["nf"] * w2 + b2
    lim["G"], lim["w2"] = abs(scale) * big(G), w2
    lim["y"] = big(X) + lim["G"] * lim["a"]
    y = X + scale * G * norm64(Fr, post)
    if pre is not None:
        lim["w1"] = big(pre.weight) if pre.weight is not None else 1.0
        b1 = big(pre.bias) if pre.bias is not None else 0.0
        lim["n_y"], lim["ny"], lim["ry"] = unit(y, pre)
        lim["h"] = lim["ny"] * lim["w1"] + b1
    return lim


def check(got, want, tol, dtype, what):
    """tol: of the fp32 computation; a bf16 result is rounded once more, by half a step (2^-8 of its value at most)."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got - want).abs()
    allowed = tol + (want.abs() * 2.0 ** -8 + tol * 2.0 ** -8 if dtype == BF16 else 0.0)
    bad = err > allowed
    assert not bad.any() and torch.isfinite(got).all(), (what, float(err.max()), float((allowed if torch.is_tensor(allowed) else torch.tensor(allowed)).max()))


def compare(x, f, gate, post, pre, act="none", scale=0.2, dim=1, seed=1, call=None, grads=("dy", "dh")):
    """One forward and backward through the public entry point against the definition."""
    dtype = x.dtype
    leaves = [t for t in (x, f, gate, *(post[1:3] if post else ()), *(pre[1:3] if pre else ())) if t is not None]
    for t in leaves:
        t.requires_grad_()
    out = (call or R().gated_residual)(x, f, post=post, gate=gate, gate_act=act, scale=scale, pre=pre, channel_dim=dim)
    y, h = out if pre is not None else (out, None)
    lim = limits(x, f, gate, post, pre, act, scale, dim)
    G = gate64(gate, x, act, dim)
    y64 = rows_of(x, dim) + scale * G * norm64(rows_of(f, dim), post)
    tol_y = 64 * U * lim["y"]
    check(rows_of(y, dim), y64, tol_y, dtype, "y")
    if h is not None:
        check(rows_of(h, dim), norm64(y64, pre), 64 * U * lim["h"] + 2 * lim["ry"] * lim["w1"] * tol_y, dtype, "h")
    g = torch.Generator().manual_seed(seed)
    give = {k: torch.randn(x.shape, generator=g).to(DEV, dtype) for k in ("dy", "dh")}
    dy = give["dy"] if "dy" in grads else None
    dh = give["dh"] if "dh" in grads and h is not None else None
    outs = [(t, d) for t, d in ((y, dy), (h, dh)) if d is not None]
    got = dict(zip(map(id, leaves), torch.autograd.grad([t for t, _ in outs], leaves, [d for _, d in outs], allow_unused=True)))
    D = rows_of(dy, dim) if dy is not None else torch.zeros_like(y64)
    tol_D = U * 2 * float(D.abs().max())
    if dh is not None:
        Y = y64.clone().requires_grad_()
        w1, b1 = (t.detach().double().cpu().requires_grad_() if t is not None else None for t in pre[1:3])
        s64 = R().NormSpec(pre.kind, w1, b1, pre.eps)
        dh64 = rows_of(dh, dim)
        zc = Y - Y.mean(1, keepdim=True) if pre.kind == "layer" else Y
        n = zc / torch.sqrt((zc * zc).mean(1, keepdim=True) + pre.eps)
        h64 = n * (w1 if w1 is not None else 1.0) + (b1 if b1 is not None else 0.0)
        need = [t for t in (Y, w1, b1) if t is not None]
        ref = dict(zip(map(id, need), torch.autograd.grad(h64, need, dh64)))
        D = D + ref[id(Y)]
        dn = float(dh64.abs().max()) * lim["w1"]
        tol_D += 64 * U * lim["ry"] * dn * (2 + lim["ny"] ** 2)
        if w1 is not None:
            check(got[id(pre.weight)], ref[id(w1)], 128 * U * ((dh64.abs() * (n.detach().abs() + lim["ny"] / 8)).sum(0)), F32, "dw_pre")
        if b1 is not None:
            check(got[id(pre.bias)], ref[id(b1)], 64 * U * dh64.abs().sum(0), F32, "db_pre")
    check(rows_of(got[id(x)], dim), D, tol_D, dtype, "dx")
    Fr = rows_of(f, dim).requires_grad_()
    w2, b2 = (t.detach().double().cpu().requires_grad_() if t is not None else None for t in (post[1:3] if post else (None, None)))
    q = gate.detach().double().cpu().requires_grad_() if gate is not None else None
    if post is not None and post.kind != "none":
        zc = Fr - Fr.mean(1, keepdim=True) if post.kind == "layer" else Fr
        n = zc / torch.sqrt((zc * zc).mean(1, keepdim=True) + post.eps)
    else:
        n = Fr
    a = n * (w2 if w2 is not None else 1.0) + (b2 if b2 is not None else 0.0)
    Gd = 1.0
    if gate is not None:
        Gd = rows_of_grad(q, dim) if gate.shape == x.shape else q.repeat_interleave(Fr.shape[0] // q.shape[0], 0) if q.dim() == 2 else q
        Gd = torch.sigmoid(Gd) if act == "sigmoid" else Gd
    u = scale * Gd * a
    need = [t for t in (Fr, q, w2, b2) if t is not None]
    ref = dict(zip(map(id, need), torch.autograd.grad(u, need, D)))
    Dmax = float(D.abs().max()) + tol_D
    slope = lim["rf"] * lim["G"] * lim["w2"] * (2 + lim["nf"] ** 2)
    check(rows_of(got[id(f)], dim), ref[id(Fr)], slope * (64 * U * Dmax + tol_D), dtype, "df")
    terms = abs(scale) * (D.abs() + tol_D / (128 * U)) if torch.is_tensor(D) else 0.0
    # tol_D stands for |D|'s own error: 128 u (|D| + tol_D / 128 u) = 128 u |D| + tol_D
    if gate is not None:
        sums = terms * (a.detach().abs() + lim["a"] / 8)
        if gate.shape == x.shape:
            check(rows_of(got[id(gate)], dim), rows_of(ref[id(q)], dim), 128 * U * sums.max(), gate.dtype, "dgate")
        elif gate.dim() == 2:
            check(got[id(gate)], ref[id(q)], 128 * U * sums.reshape(gate.shape[0], -1, gate.shape[1]).sum(1), F32, "dgate")
        else:
            check(got[id(gate)], ref[id(q)], 128 * U * sums.sum(0), F32, "dgate")
    gt = terms * (Gd.detach().abs() if torch.is_tensor(Gd) else 1.0)
    if w2 is not None:
        check(got[id(post.weight)], ref[id(w2)], 128 * U * (gt * (n.detach().abs() + lim["nf"] / 8)).sum(0), F32, "dw_post")
    if b2 is not None:
        check(got[id(post.bias)], ref[id(b2)], 128 * U * gt.sum(0), F32, "db_post")
    return y, h


def rows_of_grad(t, dim):
    return (t.movedim(1, -1) if dim == 1 else t).reshape(-1, t.shape[dim])


PLANES = [(2, 64, 8, 8), (1, 9, 5, 7), (3, 33, 1, 1), (2, 130, 9), (1, 512, 16, 16), (1, 1024, 3, 3), (2, 600, 4, 8), (1, 17, 63, 65),
          (2, 257, 2, 2), (5, 8, 1, 300), (2, 64, 64, 66), (3, 96, 7, 130)]
ROWS = [(1, 1, 512), (4, 7, 1000), (3, 50, 1024), (1, 2, 8192), (2, 300, 8), (1531, 24), (2, 5, 5001), (1, 3, 4097), (3, 2, 11, 64),
        (2, 33, 2048), (1, 700, 129), (2, 9, 8192)]
COMBOS = [("rms", "channel", "rms", "none"), ("layer", "image", "layer", "none"), ("rms", "full", "layer", "sigmoid"),
          (None, None, "rms", "none"), ("none", "channel", None, "sigmoid"), ("layer", "full", None, "none"),
          ("rms", None, "rms", "none"), ("layer", "image", "rms", "sigmoid")]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k", range(len(PLANES)))
def test_planes(k, dtype):
    for j in range(3):
        post, gate, pre, act = COMBOS[(k + 3 * j) % len(COMBOS)]
        x, f, g, p, q = make(PLANES[k], 1, dtype, post, gate, pre, seed=k + 100 * j)
        compare(x, f, g, p, q, act)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("k", range(len(ROWS)))
def test_rows(k, dtype):
    for j in range(3):
        post, gate, pre, act = COMBOS[(k + 3 * j + 1) % len(COMBOS)]
        x, f, g, p, q = make(ROWS[k], len(ROWS[k]) - 1, dtype, post, gate, pre, seed=k + 100 * j)
        compare(x, f, g, p, q, act, dim=len(ROWS[k]) - 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("combo", COMBOS)
def test_every_combination_in_both_layouts(combo, dtype):
    post, gate, pre, act = combo
    for shape, dim in (((2, 40, 6, 10), 1), ((2, 60, 40), 2)):
        for weights in (True, False):
            compare(*make(shape, dim, dtype, post, gate, pre, weights), act, scale=-0.7, dim=dim)


def test_few_channels():
    """One and three channels: a norm over so few that the layout's lanes are mostly idle (rms: with one channel the mean
    and variance form is 0 / 0 but for eps)."""
    for shape, dim in (((2, 1, 6, 6), 1), ((1, 3, 9, 8), 1), ((7, 1), 1), ((50, 3), 1), ((3, 5, 2), 2)):
        compare(*make(shape, dim, F32, "rms", "channel", "rms"), dim=dim)
    x = torch.randn(4, 1, device=DEV)
    b = torch.randn(1, device=DEV)
    assert torch.equal(R().channel_norm(x, R().NormSpec("layer", None, b)), b.expand(4, 1))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norm_alone(dtype):
    for shape, dim in (((2, 64, 8, 9), 1), ((3, 11, 1000), 2), ((2, 512, 16, 16), 1), ((6, 4096), -1)):
        for kind in ("rms", "layer"):
            g = torch.Generator().manual_seed(3)
            x = (torch.randn(shape, generator=g) + 1).to(DEV, dtype).requires_grad_()
            spec = spec_of(kind, shape[dim], True, g)
            for t in spec[1:3]:
                if t is not None:
                    t.requires_grad_()
            h = R().channel_norm(x, spec, channel_dim=dim)
            X = rows_of(x, dim).requires_grad_()
            w, b = (t.detach().double().cpu().requires_grad_() if t is not None else None for t in spec[1:3])
            zc = X - X.mean(1, keepdim=True) if kind == "layer" else X
            r = 1 / torch.sqrt((zc * zc).mean(1, keepdim=True) + spec.eps)
            n = zc * r
            h64 = n * w + (b if b is not None else 0.0)
            nmax = float((n.abs() + X.abs() * r).detach().max())
            check(rows_of(h, dim), h64.detach(), 64 * U * (nmax * float(w.detach().abs().max()) + 1), dtype, "h")
            dh = torch.randn(shape, generator=g).to(DEV, dtype)
            got = torch.autograd.grad(h, [t for t in (x, *spec[1:3]) if t is not None], dh)
            dh64 = rows_of(dh, dim)
            ref = torch.autograd.grad(h64, [t for t in (X, w, b) if t is not None], dh64)
            slope = float(r.detach().max()) * float(w.detach().abs().max()) * float(dh64.abs().max())
            check(rows_of(got[0], dim), ref[0], 64 * U * slope * (2 + nmax ** 2), dtype, "dx")
            check(got[1], ref[1], 128 * U * (dh64.abs() * (n.detach().abs() + nmax / 8)).sum(0), F32, "dw")
            if b is not None:
                check(got[2], ref[2], 64 * U * dh64.abs().sum(0), F32, "db")


def test_gradient_against_differences():
    """(L(p + e v) - L(p - e v)) / 2 e of the whole operator, L computed from its own fp32 outputs summed in 64 bits: the outputs'
    rounding is 64 u of values near 4 over 3000 elements (at most 0.03 / e relative to nothing: e = 0.01 leaves under
    1e-3 of a directional derivative of order 10), the third-order term about e^2."""
    for dim, shape in ((1, (2, 24, 6, 10)), (2, (2, 60, 24))):
        x, f, g, post, pre = make(shape, dim, F32, "layer", "full", "rms", seed=5)
        names = {"x": x, "f": f, "gate": g, "w_post": post.weight, "b_post": post.bias, "w_pre": pre.weight}
        wy, wh = (torch.randn(shape, device=DEV) for _ in range(2))

        def loss(t):
            y, h = R().gated_residual(t["x"], t["f"], post=R().NormSpec("layer", t["w_post"], t["b_post"], 1e-5), gate=t["gate"],
                                      gate_act="sigmoid", scale=0.8, pre=R().NormSpec("rms", t["w_pre"], None, 1e-5), channel_dim=dim)
            return (y.double() * wy).sum() + (h.double() * wh).sum()
        leaves = {k: t.clone().requires_grad_() for k, t in names.items()}
        grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
        for k, t in names.items():
            v = torch.sign(grads[k])                  # a direction in which the loss moves
            e = 0.01
            up, down = (loss({**names, k: t + s * e * v}) for s in (1, -1))
            want = float((up - down) / (2 * e))
            assert abs(float((grads[k] * v).sum()) / want - 1) < 2e-3, (k, dim)


def test_only_what_is_asked_for():
    """h unused, y unused, frozen leaves: the same gradients as with everything wanted, and none for the rest."""
    for shape, dim in (((2, 40, 6, 10), 1), ((2, 60, 40), 2)):
        for grads in (("dy",), ("dh",)):
            compare(*make(shape, dim, F32, "layer", "channel", "layer"), dim=dim, grads=grads)
        args = make(shape, dim, F32, "layer", "image", "layer")
        leaves = [args[0], args[1], args[2], *args[3][1:3], *args[4][1:3]]
        run = lambda: R().gated_residual(args[0], args[1], post=args[3], gate=args[2], pre=args[4], channel_dim=dim)  # noqa: E731
        dy, dh = torch.randn(shape, device=DEV), torch.randn(shape, device=DEV)
        for t in leaves:
            t.requires_grad_()
        full = torch.autograd.grad(run(), leaves, (dy, dh))
        for i, t in enumerate(leaves):
            for u in leaves:
                u.requires_grad_(u is t)
            # the sums over 120 pixels may be shared out otherwise: 64 u of the sum of their terms' magnitudes (about 1 each)
            assert float((torch.autograd.grad(run(), [t], (dy, dh))[0] - full[i]).abs().max()) <= 64 * U * 120, i
        for u in leaves:
            u.requires_grad_(False)
        assert not run()[0].requires_grad
        x = args[0].clone().requires_grad_()
        with pytest.raises(RuntimeError):       # differentiable once
            g, = torch.autograd.grad(R().channel_norm(x, args[4], dim).sum(), x, create_graph=True)
            torch.autograd.grad(g.sum(), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_orders_and_alignment(dtype):
    R_ = R()
    base = make((3, 48, 6, 8), 1, dtype, "layer", "full", "rms")
    want = R_.gated_residual(base[0], base[1], post=base[3], gate=base[2], pre=base[4])
    wide = torch.randn(3, 64, 6, 8, device=DEV).to(dtype)
    wide[:, 8:56] = base[0]
    last = lambda t: t.to(memory_format=torch.channels_last)  # noqa: E731
    odd = torch.zeros(base[1].numel() + 1, device=DEV, dtype=dtype)[1:].view(base[1].shape)
    odd.copy_(base[1])
    variants = [(wide[:, 8:56], base[1], base[2]), (base[0], odd, base[2]), (last(base[0]), last(base[1]), last(base[2])),
                (last(base[0]), base[1], odd.copy_(base[1]) if False else base[2]), (base[0], last(base[1]), base[2]),
                (base[0].transpose(2, 3).contiguous().transpose(2, 3), base[1], base[2]),
                (torch.stack([base[0], base[0]], 1)[:, 0], base[1], base[2])]
    for x, f, g in variants:
        keep = wide.clone()
        y, h = R_.gated_residual(x, f, post=base[3], gate=g, pre=base[4])
        assert torch.equal(wide, keep)
        # another order sums in another order: 64 u of values near 8 apart in fp32, a rounding step in bf16
        for a, b in ((y, want[0]), (h, want[1])):
            assert float((a.float() - b.float()).abs().max()) <= (2.0 ** -8 if dtype == BF16 else 64 * U) * 8
        if x.is_contiguous(memory_format=torch.channels_last) and not x.is_contiguous():
            assert y.is_contiguous(memory_format=torch.channels_last) and h.is_contiguous(memory_format=torch.channels_last)
    compare(last(base[0]).detach(), last(base[1]).detach(), last(base[2]).detach(), base[3], base[4], "sigmoid")
    compare(wide[:, 8:56].detach(), odd.detach(), base[2].detach(), base[3], base[4], "sigmoid")
    # rows: a slice of wider rows, an offset that breaks 16-byte alignment, batch and row dims that do not collapse
    x, f, g, post, pre = make((4, 6, 40), 2, dtype, "rms", "image", "layer")
    buf = torch.randn(4, 6, 100, device=DEV).to(dtype)
    buf[..., 8:48] = x
    off = torch.randn(4, 6, 43, device=DEV).to(dtype)
    off[..., 1:41] = f
    compare(buf[..., 8:48].detach(), off[..., 1:41].detach(), g, post, pre, dim=2)
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    compare(t.detach(), f.detach(), g.detach(), post, pre, dim=2)
    # an expanded gradient (stride 0), as sum() gives
    x = x.detach().requires_grad_()
    y = R_.gated_residual(x, f.detach(), post=post, channel_dim=2)
    y.sum().backward()
    assert torch.equal(x.grad, torch.ones_like(x))


def test_weights_and_gates_in_bf16():
    x, f, g, post, pre = make((2, 40, 6, 10), 1, BF16, "layer", "channel", "layer")
    low = lambda s: R().NormSpec(s.kind, s.weight.to(BF16).requires_grad_(), s.bias.to(BF16).requires_grad_(), s.eps)  # noqa: E731
    post, pre, g = low(post), low(pre), g.to(BF16).requires_grad_()
    up = lambda s: R().NormSpec(s.kind, s.weight.float(), s.bias.float(), s.eps)  # noqa: E731
    got = R().gated_residual(x, f, post=post, gate=g, pre=pre)
    want = R().gated_residual(x, f, post=up(post), gate=g.float(), pre=up(pre))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    grads = torch.autograd.grad(got, [post.weight, post.bias, pre.weight, pre.bias, g], (x, f))
    assert all(t.dtype == BF16 and t.shape == (40,) for t in grads)


def test_rows_that_hold_nothing_and_rows_that_are_not_numbers():
    """A row of zeros is 0 * 1 / sqrt(eps): zeros (and finite gradients); infinities and NaN stay in their own pixel."""
    for shape, dim in (((2, 40, 6, 10), 1), ((120, 40), 1)):
        x, f, g, post, pre = make(shape, dim, F32, "layer", "channel", "layer")
        clean = R().gated_residual(x, f, post=post, gate=g, pre=pre, channel_dim=dim)
        X, F_ = x.clone(), f.clone()
        xr, fr = (t.movedim(1, -1).reshape(-1, 40) for t in (X, F_))
        idx = [(3, 0.0), (7, float("inf")), (11, float("nan")), (50, 1e4)]
        for i, v in idx:
            xr[i], fr[i] = v, v
        back = lambda t: t.reshape(*shape[:1], *shape[2:], 40).movedim(-1, 1).contiguous()  # noqa: E731
        xs, fs = back(xr).requires_grad_(), back(fr).requires_grad_()
        y, h = R().gated_residual(xs, fs, post=post, gate=g, pre=pre, channel_dim=dim)
        good = torch.ones(120, dtype=torch.bool, device=DEV)
        good[[i for i, _ in idx]] = False
        for a, b in ((y, clean[0]), (h, clean[1])):
            assert torch.equal(rows_of(a, 1)[good.cpu()], rows_of(b, 1)[good.cpu()])
        h64 = rows_of(h, 1)
        assert torch.isnan(h64[7]).all() and torch.isnan(h64[11]).all() and torch.isfinite(h64[[3, 50]]).all()
        gx, gf = torch.autograd.grad((y, h), (xs, fs), (torch.ones_like(y), torch.ones_like(h)))
        assert torch.isfinite(rows_of(gx, 1)[good.cpu()]).all() and torch.isfinite(rows_of(gf, 1)[good.cpu()]).all()
        assert torch.isfinite(rows_of(gx, 1)[[3, 50]]).all() and torch.isfinite(rows_of(gf, 1)[[3, 50]]).all()


def test_empty_batches():
    for shape, dim in (((0, 40, 6, 10), 1), ((2, 40, 0, 10), 1), ((0, 40), 1), ((2, 0, 40), 2)):
        x, f = (torch.zeros(shape, device=DEV, requires_grad=True) for _ in range(2))
        post = R().NormSpec("layer", torch.ones(40, device=DEV, requires_grad=True), torch.zeros(40, device=DEV, requires_grad=True))
        gate = torch.ones(shape[0], 40, device=DEV, requires_grad=True) if len(shape) > 2 else torch.ones(40, device=DEV, requires_grad=True)
        y, h = R().gated_residual(x, f, post=post, gate=gate, pre=post, channel_dim=dim)
        assert y.shape == h.shape == shape
        for t in torch.autograd.grad((y, h), (x, f, post.weight, post.bias, gate), (y.detach(), h.detach())):
            assert not t.any() and torch.isfinite(t).all()


def test_refusals():
    R_ = R()
    x = torch.randn(2, 8, 4, 4, device=DEV)
    ok = R_.NormSpec("rms")
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        R_.channel_norm(x.half(), ok)
    with pytest.raises(ValueError, match="channel_dim"):
        R_.channel_norm(x, ok, channel_dim=4)
    with pytest.raises(ValueError, match="dim 1 or last"):
        R_.channel_norm(x, ok, channel_dim=2)
    with pytest.raises(ValueError, match="kind must be"):
        R_.channel_norm(x, R_.NormSpec("none"))
    with pytest.raises(ValueError, match="NormSpec is needed"):
        R_.channel_norm(x, None)
    with pytest.raises(ValueError, match="eps"):
        R_.channel_norm(x, R_.NormSpec("rms", eps=0.0))
    with pytest.raises(ValueError, match="weight: 8 values"):
        R_.channel_norm(x, R_.NormSpec("rms", torch.ones(7, device=DEV)))
    with pytest.raises(ValueError, match="weight: 8 values"):
        R_.channel_norm(x, R_.NormSpec("rms", torch.ones(8)))
    with pytest.raises(ValueError, match="at most 1024"):
        R_.channel_norm(torch.zeros(1, 1025, 2, device=DEV), ok)
    with pytest.raises(ValueError, match="at most 8192"):
        R_.channel_norm(torch.zeros(1, 8193, device=DEV), ok)
    with pytest.raises(ValueError, match="f: "):
        R_.gated_residual(x, x[:1])
    with pytest.raises(ValueError, match="f: "):
        R_.gated_residual(x, x.to(BF16))
    for bad in (torch.ones(7, device=DEV), torch.ones(3, 8, device=DEV), torch.ones(1, device=DEV)):
        with pytest.raises(ValueError, match="gate of shape"):
            R_.gated_residual(x, x, gate=bad)
    with pytest.raises(ValueError, match="gate"):
        R_.gated_residual(x, x, gate=x.to(BF16))
    with pytest.raises(ValueError, match="gate_act"):
        R_.gated_residual(x, x, gate=torch.ones(8, device=DEV), gate_act="relu")
    with pytest.raises(ValueError, match="scale"):
        R_.gated_residual(x, x, scale=float("inf"))


def test_streams_capture_and_repeatability():
    for shape, dim in (((2, 64, 16, 18), 1), ((2, 288, 64), 2)):
        x, f, g, post, pre = make(shape, dim, BF16, "rms", "image", "layer")
        leaves = [t.requires_grad_() for t in (x, f, g, post.weight, pre.weight, pre.bias)]
        dy, dh = (torch.randn(shape, device=DEV).to(BF16) for _ in range(2))

        def run():
            y, h = R().gated_residual(x, f, post=post, gate=g, pre=pre, channel_dim=dim)
            return [y, h, *torch.autograd.grad((y, h), leaves, (dy, dh))]
        want = [t.detach().clone() for t in run()]
        assert all(torch.equal(a, b) for a, b in zip(want, run()))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        del got
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        out = [t.detach() for t in out]
        for k in range(4):
            with torch.no_grad():
                x.copy_(make(shape, dim, BF16, "rms", "image", "layer", seed=30 + k)[0])
                g.add_(0.1)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, run())), k


def test_capture_beside_a_living_graph_of_the_same_leaves_is_refused():
    x = torch.randn(2, 64, 8, 8, device=DEV, requires_grad=True)
    spec = R().NormSpec("rms", torch.ones(64, device=DEV, requires_grad=True))
    alive = R().channel_norm(x, spec)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = x.detach() * 2              # something for the graph to hold
        with pytest.raises(RuntimeError, match="recorded before this capture"):
            R().channel_norm(x, spec)
        still = R().channel_norm(x.detach(), R().NormSpec("rms", spec.weight.detach()))       # without gradients: nothing to refuse
    graph.replay()
    assert torch.equal(still, alive) and torch.equal(z, 2 * x.detach())
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = R().channel_norm(x, spec)
        g, = torch.autograd.grad(h, [x], torch.ones_like(h))
    h = h.detach()
    graph.replay()
    want = R().channel_norm(x, spec)
    assert torch.equal(h, want) and torch.equal(g, torch.autograd.grad(want, [x], torch.ones_like(want))[0])


def _stack(kind="rms", gate="channel", seed=0):
    G = pkg("esrgan.generator")
    torch.manual_seed(seed)
    blocks = [G.ResidualDenseBlock(16, 8) for _ in range(3)]
    s = R().GatedResidualStack(blocks, 16, kind, gate, gate_act="sigmoid" if gate == "input" else "none").to(DEV)
    with torch.no_grad():
        for n, p in s.named_parameters():
            if not n.startswith("blocks"):
                p.add_(0.1 * torch.randn_like(p))
    return s


def _stack64(s, x, gates=None):
    """The stack in 64 bits on the CPU from the oracle's dense block; returns (output, parameters by name)."""
    sd = {n: p.detach().double().cpu().requires_grad_() for n, p in s.named_parameters()}

    def norm(z, which, i):
        w, b = sd[f"{which}.{i}.weight"], sd.get(f"{which}.{i}.bias")
        m = s.pre[i]
        if m.kind == "layer":
            z = z - z.mean(1, keepdim=True)
        z = z / torch.sqrt((z * z).mean(1, keepdim=True) + m.eps) * w.view(1, -1, 1, 1)
        return z if b is None else z + b.view(1, -1, 1, 1)
    x = x.detach().double().cpu()
    for i in range(len(s.blocks)):
        g = torch.sigmoid(gates[i].detach().double().cpu())[:, :, None, None] if gates is not None else sd[f"gates.{i}"].view(1, -1, 1, 1)
        x = x + s.residual_scale * g * norm(ORACLE.rdb_forward(norm(x, "pre", i), sd, f"blocks.{i}."), "post", i)
    return x, sd


@pytest.mark.parametrize("kind,gate", [("rms", "channel"), ("layer", "input")])
def test_stack_of_dense_blocks_trained_with_adamw(kind, gate):
    """As they are used together: normalised, gated dense blocks, a loss, a clipped AdamW step over all their tensors."""
    OPT = pkg("optim")
    s = _stack(kind, gate)
    x = ORACLE.hash_input("stack.x", (2, 16, 12, 20)).to(DEV)
    t = ORACLE.hash_input("stack.t", (2, 16, 12, 20)).to(DEV)
    gates = [torch.randn(2, 16, device=DEV) for _ in range(3)] if gate == "input" else None
    opt = OPT.AdamW(OPT.decay_groups(s, 0.1), lr=1e-3, max_grad_norm=0.05)
    before = {n: p.detach().double().cpu().numpy() for n, p in s.named_parameters()}
    out = s(x, gates)
    loss = ((out - t) ** 2).mean()
    loss.backward()
    ref, sd = _stack64(s, x, gates)
    assert float((out.detach().double().cpu() - ref.detach()).norm() / ref.detach().norm()) < 1e-5      # nine convolutions' fp32 sums deep
    ((ref - t.double().cpu()) ** 2).mean().backward()
    grads = {n: p.grad.detach().double().cpu() for n, p in s.named_parameters()}
    for n, g in grads.items():          # LeakyReLU'(x) flips where x is within rounding of 0: a tensor's 2-norm, not its elements
        assert float((g - sd[n].grad).norm() / sd[n].grad.norm().clamp_min(1e-30)) < 2e-3, n
    norm = opt.step()
    want = math.sqrt(sum(float(g.square().sum()) for g in grads.values()))
    assert want > 0.05 and abs(float(norm) / want - 1) < 2.0 ** -22
    for n, p in s.named_parameters():
        new, _, _ = step64(before[n], 0.0, 0.0, grads[n].numpy() * (0.05 / (want + 1e-6)), 1, 1e-3, 0.9, 0.999, 1e-8, 0.1 if p.dim() > 1 else 0.0)
        got = p.detach().double().cpu().numpy()
        assert abs(got - new).max() <= U * (3 * abs(new).max() + 24 * 1e-3), n
    with pytest.raises(ValueError, match="gates"):
        s(x, None if gate == "input" else [gates])


def test_stack_in_bf16_and_without_gradients():
    s = _stack()
    x = ORACLE.hash_input("stack.x", (2, 16, 12, 20)).to(DEV)
    for b in s.blocks:
        b.compute_dtype = BF16
    with torch.no_grad():
        out = s(x.to(BF16))
    assert out.dtype == BF16 and not out.requires_grad
    ref, _ = _stack64(s, x.to(BF16))
    # three blocks, each a few roundings of 2^-9 deep in both the branch and the stream
    assert float((out.double().cpu() - ref.detach()).norm() / ref.detach().norm()) < 2e-2


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,dim", [((200, 24, 3, 5), 1), ((65, 72, 2, 2), 1), ((130, 3, 96), 2), ((1100, 2, 20), 2), ((70, 40, 1), 1)])
def test_gates_of_many_images(shape, dim, dtype):
    """More images than one workgroup joins."""
    for k, (post, pre, act) in enumerate((("rms", "rms", "none"), ("layer", "layer", "sigmoid"))):
        x, f, g, p, q = make(shape, dim, dtype, post, "image", pre, seed=k)
        compare(x, f, g, p, q, act, dim=dim)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_expanded_tensors(dtype):
    """Rows, pixels and images of stride 0 are inputs like others."""
    cases = [((3, 5, 40), (1, 1, 40), 2), ((3, 5, 40), (3, 1, 40), 2), ((3, 5, 40), (1, 5, 40), 2), ((3, 5, 40), (3, 5, 1), 2), ((3, 5, 1), (1, 1, 1), 2),
             ((3, 5, 1), (3, 1, 1), 2), ((3, 40, 4, 6), (1, 40, 4, 6), 1), ((3, 40, 4, 6), (3, 40, 1, 1), 1), ((3, 40, 4, 6), (1, 1, 4, 6), 1),
             ((3, 40, 4, 6), (1, 40, 1, 6), 1), ((6, 40), (1, 40), 1), ((6, 40, 1, 1), (1, 40, 1, 1), 1)]
    for shape, small, dim in cases:
        spec = R().NormSpec("layer")
        x, f = torch.randn(small, device=DEV).to(dtype), torch.randn(small, device=DEV).to(dtype)
        d = torch.randn(small, device=DEV).to(dtype)
        out = []
        for wide in (lambda t: t.expand(shape), lambda t: t.expand(shape).contiguous()):
            a, b = wide(x).detach().requires_grad_(), wide(f).detach().requires_grad_()
            y, h = R().gated_residual(a, b, post=spec, gate=wide(x).detach(), pre=spec, channel_dim=dim)
            out.append([y, h, *torch.autograd.grad((y, h), (a, b), (wide(d), wide(d)))])
        assert all(torch.equal(s, t) for s, t in zip(*out)), (shape, small)


def test_capture_beside_a_living_graph_of_bf16_weights_is_refused():
    x = torch.randn(2, 64, 8, 8, device=DEV)
    spec = R().NormSpec("rms", torch.ones(64, dtype=BF16, device=DEV, requires_grad=True))
    gate = torch.ones(64, dtype=BF16, device=DEV, requires_grad=True)
    for call in (lambda: R().channel_norm(x, spec), lambda: R().gated_residual(x, x, gate=gate)):
        alive = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x * 2
            with pytest.raises(RuntimeError, match="recorded before this capture"):
                call()
        del alive


def test_two_streams_at_once():
    """Calls of different sizes on two streams share nothing."""
    sets = [make(s, 1, BF16, "rms", "image", "layer", seed=k) for k, s in enumerate(((8, 64, 32, 32), (2, 200, 40, 24)))]
    def run(k):
        x, f, g, post, pre = sets[k]
        leaves = [t.requires_grad_() for t in (x, f, g, post.weight, pre.weight, pre.bias)]
        y, h = R().gated_residual(x, f, post=post, gate=g, pre=pre)
        return [t.detach() for t in (y, h, *torch.autograd.grad((y, h), leaves, (y.detach(), h.detach())))]
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(run(k))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[k]))


def test_a_gate_of_each_row_in_fp32():
    """[B, C] in bf16 with an fp32 gate of the same shape: a gate for each of B."""
    x, f, _, post, pre = make((90, 48), 1, BF16, "rms", None, "rms")
    g = (0.5 + 0.3 * torch.randn(90, 48, generator=torch.Generator().manual_seed(7))).to(DEV)
    y, h = R().gated_residual(x, f, post=post, gate=g, pre=pre)
    want = rows_of(x, 1) + g.double().cpu() * norm64(rows_of(f, 1), post)
    lim = limits(x, f, None, post, pre, "none", float(g.abs().max()), 1)
    check(rows_of(y, 1), want, 64 * U * lim["y"], BF16, "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,dim", [((2, 20, 300, 301), 1), ((3, 99, 300, 101), 1), ((1, 5, 700, 701), 1), ((3, 40000, 40), 2), ((2, 30000, 136), 2)])
def test_more_tiles_than_workgroups(shape, dim, dtype):
    """Workgroups that take several tiles, with waves that a workgroup does not have, against the same pixels in parts."""
    for k, (post, gate, pre, act) in enumerate((("rms", "channel", "rms", "none"), ("layer", "image", "layer", "sigmoid"))):
        x, f, g, p, q = make(shape, dim, dtype, post, gate, pre, seed=k)
        leaves = [t.requires_grad_() for t in (x, f, g, *p[1:3], *q[1:3]) if t is not None]
        gen = torch.Generator().manual_seed(9)
        dy, dh = (torch.randn(shape, generator=gen).to(DEV, dtype) for _ in range(2))

        def run(x, f, g, dy, dh, leaves):
            y, h = R().gated_residual(x, f, post=p, gate=g, gate_act=act, pre=q, scale=0.2, channel_dim=dim)
            return [y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (dy, dh))]
        whole = run(x, f, g, dy, dh, leaves)
        # in parts: pixels (rows) cut into ten, images one by one, each small enough that a workgroup takes one tile
        at, cuts = (2 if dim == 1 else 1), 10
        parts = []
        for i in range(shape[0]):
            for c in range(cuts):
                piece = lambda t: t.detach()[i:i + 1].tensor_split(cuts, at)[c].contiguous()  # noqa: E731
                a, b = piece(x).requires_grad_(), piece(f).requires_grad_()
                gg = g.detach()[i:i + 1].requires_grad_() if gate == "image" else g
                parts.append((i, run(a, b, gg, piece(dy), piece(dh), [a, b, gg] + leaves[3:])))
        for k in range(4):            # y, h, dx, df: each pixel's own; the order of a sum over channels may differ
            want = torch.cat([torch.cat([r[k] for j, r in parts if j == i], at) for i in range(shape[0])])
            tol = (64 * U if dtype == F32 else 2.0 ** -7) * float(want.float().abs().max())
            assert float((whole[k].float() - want.float()).abs().max()) <= tol, k
        n = x.numel() // shape[dim]
        for k in range(4, len(whole)):
            vals = torch.stack([r[k].double().reshape(-1) for _, r in parts])
            if k == 4 and gate == "image":
                want = torch.stack([sum(r[k].double()[0] for j, r in parts if j == i) for i in range(shape[0])])
            else:
                want = vals.sum(0).view(whole[k].shape)
            # sums of n terms, each below 60 in magnitude here and with a random sign: rounding in 32 bits over chains of a
            # few hundred stays below 2^-24 * 64 of sum |term| <= 60 n
            assert float((whole[k].double() - want).abs().max()) <= 64 * U * 60 * n, k


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(3, 700, 520), (2, 1030, 1000), (1, 2049, 1024), (1, 2048, 1024), (2100, 513)])
def test_rows_enough_for_a_wave_each(shape, dtype):
    """Rows of more than 512 channels, on both sides of the number of rows from which a wave takes one by itself."""
    for k, (post, gate, pre, act) in enumerate((("rms", "channel", "rms", "none"), ("layer", None, "layer", "none"))):
        x, f, g, p, q = make(shape, len(shape) - 1, dtype, post, gate, pre, seed=k)
        compare(x, f, g, p, q, act, dim=len(shape) - 1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_many_rows_with_a_full_gate(kind, dtype):
    """Enough rows for workgroups of four waves backward, against the same rows in parts that are too few for them."""
    for rows, c in ((110000, 72), (13000, 1030)):
        x, f, g, p, q = make((rows, c), 1, dtype, kind, "full", kind, seed=rows)
        gen = torch.Generator().manual_seed(3)
        dy, dh = (torch.randn((rows, c), generator=gen).to(DEV, dtype) for _ in range(2))
        weights = [t.requires_grad_() for t in (*p[1:3], *q[1:3]) if t is not None]

        def run(*ts):
            a, b, k = (t.detach().requires_grad_() for t in ts[:3])
            y, h = R().gated_residual(a, b, post=p, gate=k, gate_act="sigmoid", pre=q, scale=0.3, channel_dim=1)
            return [y.detach(), h.detach(), *torch.autograd.grad((y, h), [a, b, k] + weights, ts[3:])]
        whole = run(x, f, g, dy, dh)
        parts = [run(*ts) for ts in zip(*(t.tensor_split(20) for t in (x, f, g, dy, dh)))]
        for k in range(5):
            want = torch.cat([r[k] for r in parts])
            tol = (64 * U if dtype == F32 else 2.0 ** -7) * float(want.float().abs().max())
            assert float((whole[k].float() - want.float()).abs().max()) <= tol, (rows, k)
        for k in range(5, len(whole)):            # sums of `rows` terms below 60 each, as above
            want = torch.stack([r[k].double() for r in parts]).sum(0)
            assert float((whole[k].double() - want).abs().max()) <= 64 * U * 60 * rows, (rows, k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(5, 64, 64, 66), (1, 130, 64, 66), (5, 300, 48, 47), (3, 1024, 40, 41), (9, 513, 18, 27), (300, 260, 5),
                                   (300, 260, 3), (260, 700, 4), (150, 40, 2), (140, 300, 7)])
def test_maps_with_two_and_four_pixels_a_thread(shape, dtype):
    for k, (post, gate, pre, act) in enumerate((("rms", "channel", "rms", "none"), ("layer", "image", "layer", "sigmoid"), ("rms", "full", "rms", "none"))):
        x, f, g, p, q = make(shape, 1, dtype, post, gate, pre, seed=k)
        compare(x, f, g, p, q, act)


@pytest.mark.parametrize("dim,shape", [(1, (3, 40, 9, 11)), (2, (3, 50, 72))])
def test_one_tensor_in_every_place(dim, shape):
    """x, f and a full gate that are one leaf, norms that share their weights: gradients add up."""
    c = shape[dim]
    gen = torch.Generator().manual_seed(4)
    t = torch.randn(shape, generator=gen).to(DEV).requires_grad_()
    w, b = ((1 + 0.1 * torch.randn(c, generator=gen)).to(DEV).requires_grad_() for _ in range(2))
    dy, dh = (torch.randn(shape, generator=gen).to(DEV) for _ in range(2))

    def run(x, f, g, w2, b2, w1, b1):
        y, h = R().gated_residual(x, f, post=R().NormSpec("layer", w2, b2), gate=g, pre=R().NormSpec("layer", w1, b1), channel_dim=dim)
        return y, h
    got = torch.autograd.grad(run(t, t, t, w, b, w, b), [t, w, b], (dy, dh))
    parts = [v.detach().clone().requires_grad_() for v in (t, t, t, w, b, w, b)]
    apart = torch.autograd.grad(run(*parts), parts, (dy, dh))
    for g, want in zip(got, (apart[0] + apart[1] + apart[2], apart[3] + apart[5], apart[4] + apart[6])):
        # the same kernels; only the order in which autograd adds two or three gradients may differ
        assert float((g - want).abs().max()) <= 3 * 2.0 ** -24 * float(sum(v.abs().max() for v in apart[:3]) if g.shape == t.shape else 2 * want.abs().max() + 100)


def test_graphs_of_two_calls_replayed_in_turn():
    """Two captured passes of one shape hold workspaces of their own."""
    sets = []
    for k in range(2):
        x, f, g, post, pre = make((4, 64, 20, 22), 1, BF16, "rms", "channel", "rms", seed=50 + k)
        leaves = [t.requires_grad_() for t in (x, f, g, post.weight, pre.weight)]
        sets.append((x, f, g, post, pre, leaves))

    def run(s):
        y, h = R().gated_residual(s[0], s[1], post=s[3], gate=s[2], pre=s[4])
        return [v.detach() for v in (y, h, *torch.autograd.grad((y, h), s[5], (s[0].detach(), s[1].detach())))]
    want = [[v.clone() for v in run(s)] for s in sets]
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(s))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for turn in range(4):
        for k in (0, 1) if turn % 2 else (1, 0):
            for v in outs[k]:
                v.zero_()
        torch.cuda.synchronize()
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        run(sets[turn % 2])
        torch.cuda.synchronize()
        for k in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k])), turn


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,dim", [((300, 64, 10, 22), 1), ((20, 64, 40, 41), 1), ((520, 8, 12, 12), 1), ((300, 40, 260), 2), ((600, 9, 70), 2)])
def test_shares_of_images_in_rounds(shape, dim, dtype):
    """Numbers of images that do not divide the workgroups: shares of one image on several, several on one."""
    x, f, g, p, q = make(shape, dim, dtype, "rms", "image", "rms", seed=3)
    compare(x, f, g, p, q, "sigmoid", dim=dim)
