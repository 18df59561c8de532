"""GPU: the AdamW step over many tensors against its definition in 64 bits, its 8-bit moments against the same operations in
numpy bit for bit, clipping, skipping, masters, state files, streams, capture, and the trainers that run it."""
import math

import numpy as np
import pytest
import torch

from helpers import O as ORACLE, pkg
from optim_ref import M_BASE, V_BASE, factor_and_norm, from8, moments32, step64, to8

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8)
F32 = torch.float32
BF16 = torch.bfloat16


def AdamW(*a, **k):
    return pkg("optim").AdamW(*a, **k)


def make(sizes, dtype=F32, seed=0, shift=0, scale=1e-2):
    """Parameters and gradients; shift: elements in front of each tensor in its storage (unaligned views)."""
    g = torch.Generator().manual_seed(seed)
    ps, gs = [], []
    for n in sizes:
        for out, mul in ((ps, 1.0), (gs, scale)):
            t = torch.zeros(n + shift, dtype=dtype, device=DEV)[shift:]
            t.copy_((mul * torch.randn(n, generator=g)).to(dtype))
            out.append(t)
    return [torch.nn.Parameter(p) for p in ps], gs


def npf(t):
    return t.detach().float().cpu().numpy().copy()


def states(opt, which):
    """One fp32 array per parameter."""
    flat = opt.moments()[which].cpu().numpy()
    return [flat[256 * f:256 * f + n].copy() for f, n in zip(opt._first, opt._n)]


def padding_is_zero(opt):
    for flat in opt.moments():
        mask = torch.ones(flat.numel(), dtype=torch.bool, device=DEV)
        for f, n in zip(opt._first, opt._n):
            mask[256 * f:256 * f + n] = False
        assert not flat[mask].any()


# Rounding of one step in fp32 (u = 2^-24): m and v take three roundings of values no larger than the largest summand, and
# inherit the error of the stored one: |dm| <= 4 u max|m| a step, the same for v.  The update is m / (sqrt(v) root + eps) times a
# constant: relative error <= 12 u from its operations plus those of m and half of v's, and p takes two roundings: 2 u |p|.
def close(got, want, upd, steps, what):
    u = 2.0 ** -24
    tol = steps * (3 * u * np.abs(want).max() + 24 * u * upd)
    err = np.abs(got - want).max() if want.size else 0.0
    assert err <= tol, (what, err, tol)


SIZES = [1, 3, 64, 255, 256, 257, 1000, 4095, 4096, 4097, 70001]


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("bits", [32, 8])
def test_three_steps_fp32(bits, shift, clip):
    ps, _ = make(SIZES, shift=shift)
    half = len(SIZES) // 2
    opt = AdamW([{"params": ps[:half], "weight_decay": 0.1}, {"params": ps[half:], "weight_decay": 0.0, "lr": 1e-3, "betas": (0.8, 0.99)}],
                state_bits=bits, max_grad_norm=clip, **HYPER)
    hyper = [(3e-3, 0.9, 0.999, 1e-8, 0.1)] * half + [(1e-3, 0.8, 0.99, 1e-8, 0.0)] * (len(SIZES) - half)
    p = [npf(x).astype(np.float64) for x in ps]
    m, v = ([np.zeros(n) for n in SIZES] for _ in range(2))
    for t in (1, 2, 3):
        _, gs = make(SIZES, seed=100 + t, shift=shift)
        norm = opt.step(gs, grad_scale=0.5)
        factor, want_norm = factor_and_norm([npf(g) for g in gs], 0.5, clip)
        if clip is None:
            assert norm is None
        else:
            assert want_norm > clip and abs(float(norm) / want_norm - 1) < 2.0 ** -23
        got_m, got_v = states(opt, 0), states(opt, 1)
        for i, (h, g) in enumerate(zip(hyper, gs)):
            lr, b1, b2, eps, wd = h
            before = p[i].copy()
            m32, v32 = moments32(m[i].astype(np.float32), v[i].astype(np.float32), npf(g), factor, b1, b2)
            p[i], m[i], v[i] = step64(p[i], m[i], v[i], npf(g).astype(np.float64) * factor, t, *h)
            close(npf(ps[i]), p[i], np.abs(p[i] - before * (1 - lr * wd)).max(), t, f"p[{i}]")
            if bits == 32:
                np.testing.assert_allclose(got_m[i], m[i], rtol=0, atol=4 * t * 2.0 ** -24 * np.abs(m[i]).max())
                np.testing.assert_allclose(got_v[i], v[i], rtol=0, atol=4 * t * 2.0 ** -24 * np.abs(v[i]).max())
            else:          # the stored moments, bit for bit; the next step goes on from them
                for got, new, base, least, signed in ((got_m[i], m32, M_BASE, 0, True), (got_v[i], v32, V_BASE, 1, False)):
                    code, scale = to8(new, base, least, signed)
                    assert np.array_equal(got, from8(code, scale, base, signed)), i
                m[i], v[i] = got_m[i].astype(np.float64), got_v[i].astype(np.float64)
            p[i] = npf(ps[i]).astype(np.float64)
    assert opt.step_counts == [3] * len(SIZES)
    padding_is_zero(opt)


@pytest.mark.parametrize("gdtype", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_bf16_parameters_move_with_their_fp32_masters(bits, gdtype):
    ps, _ = make(SIZES, BF16, shift=1)
    opt = AdamW(ps, weight_decay=0.01, state_bits=bits, **HYPER)
    master = [npf(x).astype(np.float64) for x in ps]
    m, v = ([np.zeros(n) for n in SIZES] for _ in range(2))
    for t in (1, 2, 3):
        gs = [g.to(gdtype) for g in make(SIZES, BF16, seed=t)[1]]
        opt.step(gs)
        for i, g in enumerate(gs):
            g = npf(g).astype(np.float64)
            before = master[i]
            want, m[i], v[i] = step64(before, m[i], v[i], g, t, 3e-3, 0.9, 0.999, 1e-8, 0.01)
            got = npf(opt.master[opt._master_at[i]:opt._master_at[i + 1]])
            if bits == 32:
                close(got, want, np.abs(want - before * (1 - 3e-5)).max(), t, f"master[{i}]")
            assert torch.equal(ps[i].detach().cpu(), torch.from_numpy(got).to(BF16)), i     # exactly the master's rounding
            master[i] = got.astype(np.float64) if bits == 8 else want
    # a step of 3e-3 against weights near 1 is below bf16's resolution there: the masters must have moved all the same
    assert not torch.equal(opt.master, opt.master.to(BF16).float())
    # a parameter written from outside wins over its master (where it is not what the master rounds to anyway)
    held = npf(opt.master[opt._master_at[-2]:])
    base = np.where(npf(ps[-1]) == 2.0, held, np.float32(2.0)).astype(np.float64)
    with torch.no_grad():
        ps[-1].fill_(2.0)
    zero = [torch.zeros_like(p) for p in ps]
    opt.load_moments(*(torch.zeros(256 * opt.nblocks, device=DEV) for _ in range(2)), 5, master=opt.master.clone())
    opt.step(zero)
    got = npf(opt.master[opt._master_at[-2]:])
    assert (base == 2.0).mean() > 0.9 and np.abs(got - base * (1 - 3e-5)).max() <= 2.0 ** -22


def test_8_bit_extremes():
    """Blocks of zeros, one outlier of 2^40, values below the smallest code, infinities and NaN: as the same operations do."""
    n = 256 * 5 + 17
    p = torch.nn.Parameter(torch.ones(n, device=DEV))
    g = torch.full((n,), 1e-3)
    g[:256] = 0
    g[300] = 2.0 ** 20
    g[512:768] = torch.exp2(-torch.arange(256) / 8.0) * 1e-3
    g[800], g[1030], g[1300 - 20] = float("inf"), float("nan"), 0.0
    opt = AdamW([p], state_bits=8, **HYPER)
    opt.step([g.to(DEV)])
    m, v = (states(opt, k)[0] for k in (0, 1))
    z = np.zeros(n, np.float32)
    m32, v32 = moments32(z, z, g.numpy(), 1.0, 0.9, 0.999)
    bad = np.zeros(n, bool)
    bad[768:1280] = True
    for got, new, base, least, signed in ((m, m32, M_BASE, 0, True), (v, v32, V_BASE, 1, False)):
        want = np.where(bad, 0, new).astype(np.float32)
        assert np.array_equal(got[~bad], from8(*to8(want, base, least, signed), base, signed)[~bad])
        assert np.isnan(got[bad]).all()
    assert (m[:256] == 0).all() and (v[:256] == 0).all()
    assert (v[512:768] > 0).all() and (m[512:768] == 0).any()      # the second moment never falls to zero beside a larger one
    pn = npf(p)
    assert np.isnan(pn[800]) and np.isnan(pn[1030]) and np.isfinite(np.delete(pn, [800, 1030])).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_moves_in_a_skipped_step(bits):
    ps, gs = make([300, 5000, 7])
    opt = AdamW(ps, state_bits=bits, skip_nonfinite=True, max_grad_norm=1.0, **HYPER)
    opt.step(gs)
    before = [p.detach().clone() for p in ps] + [t.clone() for t in opt.moments()]
    for bad in (float("inf"), -float("inf"), float("nan")):
        g = [x.clone() for x in gs]
        g[1][4097] = bad
        norm = opt.step(g)
        assert not math.isfinite(float(norm))
        assert all(torch.equal(a, b) for a, b in zip(before, [p.detach() for p in ps] + list(opt.moments())))
        assert opt.step_counts == [1, 1, 1]
    # squares beyond fp32's range are summed in 64 bits: this norm is a finite number, and the step is taken
    g = [x.clone() for x in gs]
    g[1][3] = 1e30
    assert abs(float(opt.step(g)) / 1e30 - 1) < 1e-6 and opt.step_counts == [2, 2, 2]
    # without skip_nonfinite a NaN goes into everything that clipping scales
    opt = AdamW(ps, max_grad_norm=1.0, **HYPER)
    g[0][0] = float("nan")
    opt.step(g)
    assert all(torch.isnan(p).all() for p in ps)


def test_a_parameter_without_gradient_stays():
    ps, gs = make([300, 5000, 7, 0])
    opt = AdamW(ps, state_bits=8, max_grad_norm=10.0, **HYPER)
    keep = ps[1].detach().clone()
    norm = opt.step([gs[0], None, gs[2], None])
    want = math.sqrt(sum(float(gs[k].double().square().sum()) for k in (0, 2)))
    assert abs(float(norm) / want - 1) < 2.0 ** -23
    assert torch.equal(ps[1], keep) and not states(opt, 0)[1].any() and opt.step_counts == [1, 0, 1, 0]
    ps[1].grad = gs[1]
    opt.step()                      # .grad of the parameters: only one has any
    assert opt.step_counts == [1, 1, 1, 0] and not torch.equal(ps[1], keep)
    opt.step([None] * 4)
    assert opt.step_counts == [1, 1, 1, 0]
    # bias corrections go by each tensor's own count: this was its first step (of at most lr = 3e-3)
    want, _, _ = step64(npf(keep).astype(np.float64), 0.0, 0.0, npf(gs[1]).astype(np.float64), 1, 3e-3, 0.9, 0.999, 1e-8, 1e-2)
    close(npf(ps[1]), want, 3e-3, 1, "first step")


@pytest.mark.parametrize("count", [449, 1000, 16400])
def test_many_tensors(count):
    """More tensors than one launch's arguments hold, more than one prepare launch's; some empty, some without gradient."""
    sizes = [k % 5 for k in range(count - 1)] + [9000]
    total = sum(sizes)
    p0, g0 = torch.randn(total, device=DEV), torch.randn(total, device=DEV)
    flat = p0.clone()
    ps, gs = [torch.nn.Parameter(x) for x in flat.split(sizes)], list(g0.split(sizes))
    opt = AdamW(ps, max_grad_norm=1.0, **HYPER)
    norm = opt.step([None if k % 7 == 3 else g for k, g in enumerate(gs)])
    mask = torch.cat([torch.full((n,), float(k % 7 != 3)) for k, n in enumerate(sizes)]).to(DEV)
    assert abs(float(norm) / float((g0 * mask).double().norm()) - 1) < 2.0 ** -23
    g = (g0 * mask).double() / float((g0 * mask).double().norm())
    want = torch.where(mask > 0, p0.double() * (1 - 3e-5) - 3e-3 * g / (g.abs() + 1e-8), p0.double())
    # the first step's update is lr g / (|g| + eps): bounded by lr, 24 roundings of it, and three of p
    assert float((flat - want).abs().max()) <= 2.0 ** -24 * (24 * 3e-3 + 3 * float(p0.abs().max()))
    wrong = [k for k, t in enumerate(opt.step_counts) if t != int(k % 7 != 3)]
    assert wrong[:5] == []


def test_flat_gradient_is_the_same_step():
    sizes = [5, 64, 4099, 3, 9000, 1]
    p0, g0 = torch.randn(sum(sizes), device=DEV), torch.randn(sum(sizes), device=DEV)
    out = []
    for way in ("list", "flat", "bf16"):
        flat = p0.clone()
        ps = [torch.nn.Parameter(x) for x in flat.split(sizes)]
        # groups in another order than the storage
        opt = AdamW([{"params": ps[3:]}, {"params": ps[:3], "weight_decay": 0.5}], state_bits=8, max_grad_norm=1.0, **HYPER)
        gs = g0.split(sizes)
        for _ in range(2):
            norm = opt.step(g0) if way == "flat" else opt.step(g0.to(BF16)) if way == "bf16" else opt.step(list(gs[3:]) + list(gs[:3]))
        out.append((flat, norm, *opt.moments()))
    assert all(torch.equal(a, b) for a, b in zip(out[0], out[1]))
    assert float((out[2][0] - out[0][0]).abs().max()) < 2e-3            # bf16 gradients: another step, but near
    apart = [torch.nn.Parameter(torch.randn(4, device=DEV)) for _ in range(2)]
    gap = [torch.nn.Parameter(x) for x in torch.randn(12, device=DEV).split(4)][::2]
    for ps in (apart, gap):
        if ps is gap or apart[1].data_ptr() - apart[0].data_ptr() != 16:
            with pytest.raises(ValueError, match="covering one flat buffer"):
                AdamW(ps).step(torch.zeros(8, device=DEV))
    with pytest.raises(ValueError, match="flat gradient"):
        opt.step(torch.zeros(3, device=DEV))


def test_gradients_in_other_layouts_and_types():
    p = torch.nn.Parameter(torch.randn(6, 50, device=DEV))
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn(50, 6, device=DEV).t()
    a, b = AdamW([p]), AdamW([q])
    a.step([g])
    b.step([g.contiguous()])
    assert torch.equal(p, q)
    with pytest.raises(ValueError, match="gradient 0 has shape"):
        a.step([torch.zeros(50, 6, device=DEV)])
    with pytest.raises(ValueError, match="gradient 0 has shape"):
        a.step([torch.zeros(6, 50)])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        a.step([torch.zeros(6, 50, device=DEV, dtype=torch.float16)])
    with pytest.raises(ValueError, match="1 gradients for|2 gradients for"):
        a.step([g, g])
    with pytest.raises(ValueError, match="grad_scale"):
        a.step([g], grad_scale=float("nan"))
    a.param_groups[0]["lr"] = -1.0
    with pytest.raises(ValueError, match="lr, eps and weight_decay"):
        a.step([g])


def test_refused_parameters():
    x = torch.randn(64, device=DEV)
    p = torch.nn.Parameter(x)
    with pytest.raises(ValueError, match="given twice|share memory"):
        AdamW([p, p])
    with pytest.raises(ValueError, match="share memory"):
        AdamW([x[:40], x[39:]])
    with pytest.raises(ValueError, match="not contiguous"):
        AdamW([x.view(8, 8).t()])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        AdamW([x.half()])
    AdamW([x[:40], x[40:]])


def test_follows_parameters_to_new_storage():
    G = pkg("esrgan.generator")
    flatten = pkg("utils.flat").flatten_parameters
    gen = G.GeneratorESRGAN(num_features=16, num_blocks=1).to(DEV)
    opt = AdamW(pkg("optim").decay_groups(gen))
    old = [p.data for p in gen.parameters()]
    keep = [t.clone() for t in old]
    flat = flatten(gen)
    opt.step([torch.ones_like(p) for p in opt.params])
    assert all(torch.equal(a, b) for a, b in zip(old, keep))             # the old storage is not touched any more
    assert not torch.equal(flat, torch.cat([t.reshape(-1) for t in keep]))
    opt.step(torch.ones_like(flat))
    gen.to(BF16)
    with pytest.raises(RuntimeError, match="build a new optimizer"):
        opt.step([torch.ones_like(p) for p in opt.params])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_and_torch_interchange(bits):
    ps, _ = make(SIZES)
    pb, _ = make([300, 9], BF16, seed=3)
    groups = lambda a, b: [{"params": a, "weight_decay": 0.1}, {"params": b, "lr": 1e-3}]  # noqa: E731
    opt = AdamW(groups(ps, pb), state_bits=bits, **HYPER)
    for t in range(2):
        opt.step(make(SIZES, seed=t)[1] + make([300, 9], BF16, seed=t)[1])
    sd = opt.state_dict()
    qs, qb = [torch.nn.Parameter(p.detach().clone()) for p in ps], [torch.nn.Parameter(p.detach().clone()) for p in pb]
    again = AdamW(groups(qs, qb), state_bits=bits)
    again.load_state_dict(sd)
    assert again.step_counts == opt.step_counts and again.lr == opt.lr and torch.equal(again.master, opt.master)
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), again.moments()))
    if bits == 8:        # the same codes and scales, not only the same values
        assert torch.equal(opt._m, again._m) and torch.equal(opt._v, again._v) and torch.equal(opt._m_scale, again._m_scale)
    gs = make(SIZES, seed=9)[1] + make([300, 9], BF16, seed=9)[1]
    opt.step(gs)
    again.step(gs)
    assert all(torch.equal(a, b) for a, b in zip(ps + pb, qs + qb))
    # torch's own AdamW over the fp32 tensors goes on from the file, and the other way round
    ref = torch.optim.AdamW([{"params": [torch.nn.Parameter(p.detach().clone()) for p in ps]}])
    solo = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=bits, **HYPER)
    solo.step(make(SIZES, seed=1)[1])
    ref.load_state_dict(solo.state_dict())
    for p, q in zip(ref.param_groups[0]["params"], solo.params):
        p.data.copy_(q.data)
    gs = make(SIZES, seed=2)[1]
    for p, g in zip(ref.param_groups[0]["params"], gs):
        p.grad = g
    ref.step()
    solo.step(gs)
    for p, q in zip(ref.param_groups[0]["params"], solo.params):
        # both within their own rounding of the same step: 3 u |p| + 24 u |update| each
        assert float((p - q).detach().abs().max()) <= 2.0 ** -23 * (3 * float(p.detach().abs().max()) + 24 * 0.05)
    back = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=bits)
    back.load_state_dict(ref.state_dict())
    assert back.step_counts == [2] * len(SIZES)
    with pytest.raises(ValueError, match="does not match"):
        back.load_state_dict(AdamW(ps[:2]).state_dict())


def test_another_stream_and_capture():
    ps, gs = make([300, 5000, 64], seed=1)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, ref = (AdamW(x, state_bits=8, max_grad_norm=0.1, skip_nonfinite=True, **HYPER) for x in (ps, qs))
    static = [g.clone() for g in gs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step(static)
    torch.cuda.current_stream().wait_stream(side)
    ref.step(gs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(static)
    assert opt.step_counts == [1, 1, 1]                     # capturing runs nothing
    for k in range(4):
        new = make([300, 5000, 64], seed=20 + k)[1]
        if k == 2:
            new[0][5] = float("inf")                        # skipped inside the graph as outside
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = ref.step(new)
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(a, b) for a, b in zip(ps, qs))
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), ref.moments()))
    assert opt.step_counts == ref.step_counts == [4, 4, 4]


def test_deterministic():
    out = []
    for _ in range(2):
        ps, gs = make([300000, 4097, 12345], seed=4)
        opt = AdamW(ps, state_bits=8, max_grad_norm=0.01, **HYPER)
        for _ in range(3):
            norm = opt.step(gs)
        out.append([p.detach().clone() for p in ps] + [norm.clone(), *opt.moments()])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_a_tensor_of_more_than_2_to_the_31_elements():
    n = 2 ** 31 + 4097
    p = torch.nn.Parameter(torch.ones(n, dtype=BF16, device=DEV), requires_grad=False)
    g = torch.zeros(n, dtype=BF16, device=DEV)
    g[-3:] = torch.tensor([1.0, -1.0, 0.5])
    g[5] = 1.0
    opt = AdamW([p], lr=0.25, weight_decay=0.0, state_bits=8, max_grad_norm=100.0)
    assert abs(float(opt.step([g])) - math.sqrt(3.25)) < 1e-6
    assert p[-5:].tolist() == [1.0, 1.0, 0.75, 1.25, 0.75] and p[:7].tolist() == [1, 1, 1, 1, 1, 0.75, 1]
    assert float((p == 1).sum(dtype=torch.int64)) == n - 4


def _trainer(optimizer, seed=5):
    T, G = pkg("train"), pkg("esrgan.generator")
    torch.manual_seed(0)
    gen = G.GeneratorESRGAN(num_blocks=1).to(DEV)
    tr = T.GeneratorWarmupTrainer(gen, (2, 3, 16, 16), torch.float32, optimizer=optimizer)
    lr = ORACLE.hash_input("optim.lr", (2, 3, 16, 16)).to(DEV)
    hr = ORACLE.hash_input("optim.hr", (2, 3, 64, 64)).to(DEV)
    return tr, gen, lr, hr


@pytest.mark.parametrize("bits", [32, 8])
def test_warmup_trainer_steps_with_it(bits):
    OPT = pkg("optim")
    tr, gen, lr, hr = _trainer(lambda m: OPT.AdamW(OPT.decay_groups(m, 0.1), lr=1e-3, state_bits=bits, max_grad_norm=1e-3))
    before = {n: p.detach().double().cpu().numpy() for n, p in gen.named_parameters()}
    tr.step(lr, hr)
    grads = {n: g.detach().double().cpu().numpy() for n, g in tr.plan.grads.items()}
    norm = math.sqrt(sum(float((g ** 2).sum()) for g in grads.values()))
    assert norm > 1e-3
    for n, p in gen.named_parameters():
        wd = 0.1 if p.dim() > 1 else 0.0
        g = grads[n] * (1e-3 / (norm + 1e-6))
        want, _, _ = step64(before[n], 0.0, 0.0, g, 1, 1e-3, 0.9, 0.999, 1e-8, wd)
        close(p.detach().cpu().numpy(), want, 1e-3, 1, n)
    tr.opt.lr = 0.0
    keep = tr.flat.clone()
    tr.step(lr, hr)
    assert torch.equal(tr.flat, keep)
    with pytest.raises(ValueError, match="every parameter"):
        _trainer(lambda m: OPT.AdamW([m.conv_first.weight]))


def test_training_checkpoint_with_8_bit_moments(tmp_path):
    OPT, ck = pkg("optim"), pkg("utils.checkpointing")
    mk = lambda m: OPT.AdamW(OPT.decay_groups(m, 0.1), lr=1e-3, state_bits=8)  # noqa: E731
    tr, gen, lr, hr = _trainer(mk)
    for _ in range(2):
        tr.step(lr, hr)
    ck.save_checkpoints(gen, tr.opt, 3, 0.0, 1.0, tmp_path)
    tr2, gen2, _, _ = _trainer(mk)
    assert ck.load_latest_checkpoint(gen2, tr2.opt, tmp_path) == 4
    assert torch.equal(tr2.flat, tr.flat) and torch.equal(tr2.opt._m, tr.opt._m) and torch.equal(tr2.opt._v, tr.opt._v)
    assert tr2.opt.step_counts == tr.opt.step_counts


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("flat", [False, True])
def test_a_small_step_in_one_launch_is_the_step(bits, flat):
    """The same tensors beside one that makes the step large, and by themselves: same bits; captured and replayed too."""
    sizes = [300, 0, 5000, 7, 64]
    ps, gs = make(sizes, seed=3)
    if flat:
        buf, grad = torch.cat([p.detach() for p in ps]), torch.cat(gs)
        ps, gs = [torch.nn.Parameter(x) for x in buf.split(sizes)], list(grad.split(sizes))
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    small = AdamW(ps, state_bits=bits, **HYPER)
    large = AdamW(qs + [torch.zeros(64 * 4096, device=DEV)], state_bits=bits, **HYPER)
    given = lambda k: [None if (k % 2 and i == 2) and not flat else g for i, g in enumerate(gs)]  # noqa: E731
    call = lambda k: small.step(grad if flat else given(k))  # noqa: E731
    for k in range(3):
        call(k)
        large.step(given(k) + [torch.zeros(64 * 4096, device=DEV)])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(3)
        call(4)
    for k in range(3):
        for t in gs:
            t.mul_(-0.5)
        graph.replay()
        for j in (3, 4):
            large.step(given(j) + [torch.zeros(64 * 4096, device=DEV)])
        torch.cuda.synchronize()
    assert small.step_counts == large.step_counts[:5] == ([9] * 5 if flat else [9, 9, 5, 9, 9])
    assert all(torch.equal(a, b) for a, b in zip(ps, qs))
    for a, b in zip(small.moments(), large.moments()):
        assert torch.equal(a, b[:a.numel()])


def test_addresses_left_by_the_norm_pass():
    """More tensors than one launch's addresses, of both types, some without a gradient, which change from step to step."""
    g = torch.Generator().manual_seed(2)
    sizes = [1 + int(k) for k in torch.randint(0, 700, (1000,), generator=g)]
    ps, gs = make(sizes, seed=6)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, ref = AdamW(ps, max_grad_norm=1e9, **HYPER), AdamW(qs, **HYPER)          # a norm that never clips against none
    for step in range(3):
        give = [None if (k + step) % 5 == 0 else x.to(BF16) if (k + step) % 3 == 0 else x.clone() for k, x in enumerate(gs)]
        opt.step(give)
        ref.step(give)
        del give
    assert all(torch.equal(a, b) for a, b in zip(ps, qs)) and opt.step_counts == ref.step_counts
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), ref.moments()))


def test_a_parameter_that_changed_in_place_is_seen():
    """Same address, other size, order or type: what the tables hold no longer describes it."""
    for change, error in ((lambda t: t[:40], RuntimeError), (lambda t: t.view(BF16)[:64], RuntimeError),
                          (lambda t: t.view(8, 8).t(), ValueError)):
        for grads in (lambda p: [torch.ones_like(p)], lambda p: torch.ones(p.numel(), device=DEV)):
            p = torch.nn.Parameter(torch.zeros(64, device=DEV))
            opt = AdamW([p])
            p.data = change(p.data)
            with pytest.raises(error, match="build a new optimizer|not contiguous"):
                opt.step(grads(p))
            assert not p.any()


def test_state_of_other_shapes_is_refused():
    p = torch.nn.Parameter(torch.zeros(64, dtype=BF16, device=DEV))
    opt = AdamW([p])
    opt.step([torch.ones_like(p)])
    for key in ("exp_avg", "exp_avg_sq", "master"):
        sd = opt.state_dict()
        sd["state"][0][key] = torch.zeros(1, device=DEV)
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(sd)


def test_two_optimizers_on_two_streams():
    streams, out = [torch.cuda.Stream() for _ in range(2)], []
    for where in (None, streams):
        sets = [make([30000, 77, 4096], seed=k) for k in range(2)]
        opts = [AdamW(ps, state_bits=8, max_grad_norm=0.5, **HYPER) for ps, _ in sets]
        torch.cuda.synchronize()
        for _ in range(20):
            for k in range(2):
                with torch.cuda.stream(where[k] if where else torch.cuda.current_stream()):
                    opts[k].step(sets[k][1])
        torch.cuda.synchronize()
        out.append([p.detach().clone() for ps, _ in sets for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_adversarial_trainer_steps_both_networks_with_it():
    OPT, T = pkg("optim"), pkg("train")
    torch.manual_seed(0)
    gen = pkg("esrgan.generator").GeneratorESRGAN(num_blocks=1).to(DEV)
    disc = pkg("esrgan.discriminator").Discriminator().to(DEV)
    with pytest.warns(UserWarning):
        vgg = pkg("utils.loss").VGGLoss(device=DEV, allow_synthetic=True)
    built = []

    def mk(module):
        built.append(OPT.AdamW(OPT.decay_groups(module, 0.1), lr=1e-3, state_bits=8, max_grad_norm=1.0))
        return built[-1]
    tr = T.AdversarialTrainer(gen, disc, vgg, (2, 3, 16, 16), optimizer=mk)
    assert built == [tr.opt_g, tr.opt_d]
    lr = ORACLE.hash_input("optim.lr", (2, 3, 16, 16)).to(DEV)
    hr = ORACLE.hash_input("optim.hr", (2, 3, 64, 64)).to(DEV)
    before = [tr.flat_g.clone(), tr.flat_d.clone()]
    for _ in range(2):
        tr.step(lr, hr)
    assert set(tr.opt_g.step_counts) == set(tr.opt_d.step_counts) == {2}
    for a, b in zip(before, (tr.flat_g, tr.flat_d)):
        # two steps of lr = 1e-3 that move each value by at most about lr / sqrt(1 - b2) ... * (1 - b1) each, and decay 1e-4
        assert not torch.equal(a, b) and torch.isfinite(b).all() and float((a - b).abs().max()) < 2 * 1e-3 * 3.2 + 2e-4 * float(a.abs().max())


@pytest.mark.parametrize("count", [460, 950])
@pytest.mark.parametrize("clip", [None, 1e9])
def test_gradients_far_apart(count, clip):
    """Gradients more than 2^32 elements apart at addresses that share no alignment, against gradients side by side."""
    sizes = [1 + k % 7 for k in range(count)]
    ps, gs = make(sizes, seed=8)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    space = torch.empty((1 << 32) + (1 << 20), device=DEV)
    far, at = [], 1
    for k, g in enumerate(gs):
        lo = at if k % 2 else at + (1 << 32)
        far.append(space[lo:lo + g.numel()])
        far[-1].copy_(g)
        at += g.numel()
    give = lambda xs: [None if k % 11 == 5 else x for k, x in enumerate(xs)]  # noqa: E731
    a, b = AdamW(ps, max_grad_norm=clip, **HYPER), AdamW(qs, max_grad_norm=clip, **HYPER)
    for _ in range(2):
        n, m = a.step(give(far)), b.step(give(gs))
        assert clip is None or torch.equal(n, m)
    assert all(torch.equal(x, y) for x, y in zip(ps, qs)) and a.step_counts == b.step_counts


@pytest.mark.parametrize("bits", [32, 8])
def test_scalars_and_odd_shapes(bits):
    shapes = [(), (1,), (3, 1, 5), (0, 4), (257,)]
    ps = [torch.nn.Parameter(torch.full(s, 2.0, device=DEV)) for s in shapes]
    for p in ps:
        p.grad = torch.full(p.shape, 0.25, device=DEV)
    opt = AdamW(ps, lr=0.125, weight_decay=0.0, state_bits=bits, eps=0.0)
    opt.step()
    # a first step: m / (1 - b1) = g, sqrt(v / (1 - b2)) = |g|: lr g / |g|, off by the roundings of ten operations on it
    assert all(float((p.detach() - 1.875).abs().max()) <= 0.125 * 12 * 2.0 ** -23 + 2.0 ** -23 for p in ps if p.numel())
    sd = opt.state_dict()
    assert [tuple(sd["state"][k]["exp_avg"].shape) for k in range(5)] == shapes
    other = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=0.125, weight_decay=0.0, state_bits=bits, eps=0.0)
    other.load_state_dict(sd)
    for p, q in zip(ps, other.params):
        q.grad = p.grad
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, other.params)) and other.step_counts == opt.step_counts == [2] * 5
