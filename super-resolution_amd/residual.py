"""Norms over the channels around a gated residual branch (``srx_resnorm_forward`` / ``srx_resnorm_backward``).

The reference adds a branch scaled by a constant (``x5 * 0.2 + x``, ``out * 0.2 + x``; esrgan/generator.py:23,37) and has
no norm.  :func:`gated_residual` is that add with a norm after the branch, a gate on it and the norm in front of the next
branch, in one pass over the data, forward and backward::

    y = x + scale * act(gate) * N_post(f)          h = N_pre(y)

:func:`channel_norm` is the norm alone (in front of the first branch).  ``ChannelNorm`` holds one norm's parameters,
``GatedResidualStack`` chains branches (this package's dense blocks, or any module that keeps its input's shape).

Tensors: float32 or bfloat16 on a GPU, channels at dim 1 (``[B, C, ...]`` maps, ``channel_dim=1``) or last (tokens,
``channel_dim=-1``); at most 1024 channels in maps, 8192 in channels-last tensors.  Memory order is kept: a
channels-last map gives channels-last results.  Statistics and sums are float32 whatever the type.
"""
from __future__ import annotations

import ctypes as C
import math
import weakref
from typing import NamedTuple, Optional, Sequence

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import engine

KINDS = {"none": 0, "rms": 1, "layer": 2}
ACTS = {"none": 0, "sigmoid": 1}
_DTYPE_ID = {torch.bfloat16: L.BF16, torch.float32: L.F32}


class NormSpec(NamedTuple):
    """One norm over the channels: ``kind`` "rms" (z / sqrt(mean z^2 + eps)) or "layer" ((z - mean) / sqrt(var + eps)), times
    ``weight`` plus ``bias`` ([C] each, None: 1 and 0)."""
    kind: str
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-6


class _Geometry:
    """How the channels and pixels of one call lie in memory; every tensor of the call is brought to it."""

    def __init__(self, x: torch.Tensor, channel_dim: int):
        if x.device.type != "cuda":
            raise RuntimeError(f"libsrx runs on a ROCm GPU only (input is on {x.device})")
        if x.dtype not in _DTYPE_ID:
            raise TypeError(f"float32 or bfloat16 tensors are supported, got {x.dtype}")
        dims = x.dim()
        if dims < 2 or not -dims <= channel_dim < dims:
            raise ValueError(f"channel_dim {channel_dim} of a tensor of shape {tuple(x.shape)}")
        at = channel_dim % dims
        if at not in (1, dims - 1):
            raise ValueError(f"channels must be at dim 1 or last, not at dim {at} of {dims}")
        self.shape, self.dtype, self.device = x.shape, x.dtype, x.device
        self.B, self.C = x.shape[0], x.shape[at]
        self.P = math.prod(x.shape[1:]) // self.C if self.C else 0
        # channels at dim 1 that lie innermost in memory (channels-last maps), or a single pixel: rows
        self.moved = at != dims - 1 and (self.P == 1 or (not x.is_contiguous() and x.movedim(1, -1).is_contiguous()))
        self.rows = at == dims - 1 or self.moved
        if self.C == 0:
            raise ValueError(f"no channels in a tensor of shape {tuple(x.shape)}")
        if self.C > L.RESNORM_MAX_C[int(self.rows)]:
            raise ValueError(f"{self.C} channels: at most {L.RESNORM_MAX_C[int(self.rows)]} are supported "
                             f"{'channels last' if self.rows else 'in maps'}")
        if self.B >= 2 ** 31 or self.P >= 2 ** 31:
            raise ValueError(f"sizes of 2^31 and more are not supported: {tuple(x.shape)}")

    def check(self, t: torch.Tensor, what: str) -> None:
        if t.shape != self.shape or t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"{what}: {self.dtype} of shape {tuple(self.shape)} on {self.device} expected, got {t.dtype} of "
                             f"{tuple(t.shape)} on {t.device}")

    def take(self, t: torch.Tensor):
        """(tensor that owns the memory, stride): t itself where its order fits, else a copy."""
        if self.rows:
            v = t.movedim(1, -1) if self.moved else t
            if not v.is_contiguous():
                try:
                    flat = v.view(-1, self.C)             # one stride between rows?
                    if self.C == 1 or flat.stride(1) == 1:
                        return flat, (flat.stride(0) if flat.shape[0] > 1 else self.C)
                except RuntimeError:
                    pass
                v = v.contiguous()
            return v, self.C
        n = self.C * self.P
        if not t.is_contiguous():
            inner, expect = True, n
            for size, stride in zip(t.shape[1:], t.stride()[1:]):
                expect //= max(size, 1)
                inner = inner and (size == 1 or stride == expect)
            if inner:
                return t, (t.stride(0) if self.B > 1 else n)
            t = t.contiguous()
        return t, n

    def empty(self, like: Optional[torch.Tensor] = None) -> torch.Tensor:
        """A new tensor in this order, as the caller sees it; like: a tensor of this shape and type, to copy the order of where it
        fits (half the host time of a fresh description)."""
        if like is not None and not self.moved and like.is_contiguous():
            return torch.empty_like(like)
        if self.moved:
            return torch.empty(self.shape[:1] + self.shape[2:] + self.shape[1:2], dtype=self.dtype, device=self.device).movedim(-1, 1)
        return torch.empty(self.shape, dtype=self.dtype, device=self.device)

    def out_stride(self) -> int:
        return self.C if self.rows else self.C * self.P


class _Call:
    """The plain values of one gated_residual / channel_norm call."""

    def __init__(self, geo: _Geometry, post: Optional[NormSpec], pre: Optional[NormSpec], gate_mode: int, gate_act: int, scale: float,
                 branch: bool):
        self.geo, self.gate_mode, self.branch = geo, gate_mode, branch
        d = self.desc = L.ResnormDesc()
        d.dtype, d.layout = _DTYPE_ID[geo.dtype], (L.RESNORM_ROWS if geo.rows else L.RESNORM_PLANES)
        d.B, d.C, d.P = geo.B, geo.C, geo.P
        d.post_kind = KINDS[post.kind] if post is not None else 0
        d.pre_kind = KINDS[pre.kind] if pre is not None else 0
        d.post_eps = post.eps if post is not None else 1.0
        d.pre_eps = pre.eps if pre is not None else 1.0
        d.gate_mode, d.gate_act, d.scale = gate_mode, gate_act, scale

    def fresh(self):
        d = L.ResnormDesc()
        C.memmove(C.byref(d), C.byref(self.desc), C.sizeof(d))
        return d

    def put(self, d, keep, name: str, t: Optional[torch.Tensor]) -> None:
        if t is not None:
            t, stride = self.geo.take(t)
            keep.append(t)
            setattr(d, name, t.data_ptr() or 16)       # an empty tensor has no address; nothing is read from this one
            setattr(d, name + "_stride", stride)

    def common(self, d, keep, gate, w_post, b_post, w_pre, b_pre) -> None:
        if self.gate_mode == 3:
            self.put(d, keep, "gate", gate)
        elif gate is not None:
            d.gate = gate.data_ptr() or 16
        d.w_post = w_post.data_ptr() if w_post is not None else None
        d.b_post = b_post.data_ptr() if b_post is not None else None
        d.w_pre = w_pre.data_ptr() if w_pre is not None else None
        d.b_pre = b_pre.data_ptr() if b_pre is not None else None

    def launch(self, name: str, d) -> None:
        index = self.geo.device.index
        if torch.cuda.current_device() != index:
            with torch.cuda.device(index):
                return self.launch(name, d)
        L.check(getattr(L.lib(), name)(C.byref(d), torch.cuda.current_stream().cuda_stream), name)

    def forward(self, x, f, gate, w_post, b_post, w_pre, b_pre):
        d, keep, geo = self.fresh(), [], self.geo
        self.put(d, keep, "x", x)
        self.put(d, keep, "f", f)
        self.common(d, keep, gate, w_post, b_post, w_pre, b_pre)
        y = h = None
        if f is not None:
            y = geo.empty(x)
            d.y, d.y_stride = y.data_ptr() or 16, geo.out_stride()
        if d.pre_kind:
            h = geo.empty(x)
            d.h, d.h_stride = h.data_ptr() or 16, geo.out_stride()
        self.launch("srx_resnorm_forward", d)
        return y, h


# Graphs of this module's operators that were recorded outside of a capture and still live.
_EAGER: "weakref.WeakSet" = weakref.WeakSet()


def _note_graph(ctx, tensors, device) -> None:
    """Autograd keeps one accumulator per leaf for as long as any graph of that leaf lives, bound to the stream it was
    first used on.  A backward pass captured on another stream would then make the capture wait for that stream, and
    ROCm's runtime ends the process when such a capture closes.  So the forward call is refused instead."""
    leaves = [id(t) for t in tensors if t is not None and t.is_leaf and t.requires_grad]
    if leaves:
        stream = engine.stream_ptr(device)
        if not torch.cuda.is_current_stream_capturing():
            ctx.srx_leaves, ctx.srx_stream = leaves, stream
            _EAGER.add(ctx)
        elif any(g.srx_stream != stream and not set(leaves).isdisjoint(g.srx_leaves) for g in list(_EAGER)):
            raise RuntimeError("a graph that was recorded before this capture, on another stream, still holds one of these leaves "
                               "(an output of an earlier call is alive): delete it, or capture on the stream that it was recorded on")


class _ResNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, x, f, gate, w_post, b_post, w_pre, b_pre):
        _note_graph(ctx, (x, f, gate, w_post, b_post, w_pre, b_pre), call.geo.device)
        y, h = call.forward(x, f, gate, w_post, b_post, w_pre, b_pre)
        ctx.call = call
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if h is not None else None, f, gate, w_post, b_post, w_pre, b_pre)
        return h if f is None else y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        call, geo = ctx.call, ctx.call.geo
        x, f, gate, w_post, b_post, w_pre, b_pre = ctx.saved_tensors
        dy = grads[0] if call.branch else None
        dh = grads[-1] if call.desc.pre_kind else None
        if dy is None and dh is None:
            return (None,) * 8
        _, nx, nf, ng, nwp, nbp, nw, nb = ctx.needs_input_grad
        d, keep, out = call.fresh(), [], [None] * 8
        nw, nb = nw and dh is not None, nb and dh is not None

        def new(at, name, t, stride=0):
            out[at] = t
            setattr(d, name, t.data_ptr())
            if stride:
                setattr(d, name + "_stride", stride)

        like, stride = f if f is not None else x, geo.out_stride()
        if nx:
            if dh is not None:
                new(1, "dx", geo.empty(like), stride)
            else:
                out[1] = dy                                               # without h, y's gradient is x's
        if nf:
            new(2, "df", geo.empty(like), stride)
        if ng and call.gate_mode != 1:
            new(3, "dgate", geo.empty(like) if call.gate_mode == 3 else torch.empty_like(gate), stride if call.gate_mode == 3 else 0)
        vectors = [(at, name) for at, name, need in ((3, "dgate", ng and call.gate_mode == 1), (4, "dw_post", nwp), (5, "db_post", nbp),
                                                     (6, "dw_pre", nw), (7, "db_pre", nb)) if need]
        if vectors:
            rows = torch.empty((len(vectors), geo.C), dtype=torch.float32, device=geo.device)
            for (at, name), t in zip(vectors, rows.unbind()):
                new(at, name, t)
        if nf or ng or nwp or nbp or dh is not None:
            call.put(d, keep, "x", x if dh is not None else None)
            call.put(d, keep, "f", f)                 # y is formed again from x and f
            call.common(d, keep, gate, w_post, b_post, w_pre, b_pre)
            if dh is None:
                d.pre_kind = 0
            call.put(d, keep, "dy", dy)
            call.put(d, keep, "dh", dh)
            ws = torch.empty(max(1, L.lib().srx_resnorm_ws_floats(C.byref(d))), dtype=torch.float32, device=geo.device)
            d.ws = ws.data_ptr()
            call.launch("srx_resnorm_backward", d)
        return tuple(out)


def _channel_vector(t: Optional[torch.Tensor], geo: _Geometry, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.shape != (geo.C,) or t.device != geo.device or not t.is_floating_point():
        raise ValueError(f"{what}: {geo.C} values on {geo.device} expected, got {t.dtype} of shape {tuple(t.shape)} on {t.device}")
    return t.float().contiguous()


def _checked_spec(spec: Optional[NormSpec], geo: _Geometry, what: str, least: int = 1) -> None:
    if spec is None:
        return
    if spec.kind not in KINDS or KINDS[spec.kind] < least:
        raise ValueError(f"{what}: kind must be one of {[k for k, v in KINDS.items() if v >= least]}, got {spec.kind!r}")
    if not 0 < spec.eps < math.inf:
        raise ValueError(f"{what}: eps must be positive, got {spec.eps}")


def _run(geo, x, f, gate, gate_mode, gate_act, scale, post, pre):
    w_post, b_post = (_channel_vector(post.weight, geo, "post.weight"), _channel_vector(post.bias, geo, "post.bias")) if post is not None else (None, None)
    w_pre, b_pre = (_channel_vector(pre.weight, geo, "pre.weight"), _channel_vector(pre.bias, geo, "pre.bias")) if pre is not None else (None, None)
    call = _Call(geo, post, pre, gate_mode, gate_act, scale, f is not None)
    tensors = (x, f, gate, w_post, b_post, w_pre, b_pre)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return _ResNormFn.apply(call, *tensors)
    y, h = call.forward(*tensors)
    return h if f is None else y if h is None else (y, h)


def channel_norm(x: torch.Tensor, norm: NormSpec, channel_dim: int = 1) -> torch.Tensor:
    """The norm of every pixel (row) of x over its channels."""
    geo = _Geometry(x, channel_dim)
    if norm is None:
        raise ValueError("norm: a NormSpec is needed")
    _checked_spec(norm, geo, "norm")
    return _run(geo, x, None, None, 0, 0, 1.0, None, norm)


def gated_residual(x: torch.Tensor, f: torch.Tensor, *, post: Optional[NormSpec] = None, gate: Optional[torch.Tensor] = None,
                   gate_act: str = "none", scale: float = 1.0, pre: Optional[NormSpec] = None, channel_dim: int = 1):
    """``y = x + scale * act(gate) * N_post(f)``; with ``pre`` also ``h = N_pre(y)``: returns y, or (y, h).

    x, f: same shape, type and device.  post: the norm after the branch (None: none; kind "none": only its weight and
    bias).  gate: None, [C], [B, C] (B = x.shape[0]: one gate for each image or sequence) or a tensor like f; gate_act
    "none" or "sigmoid".  pre: the norm in front of the next branch.  Differentiable once, in everything but scale and eps."""
    geo = _Geometry(x, channel_dim)
    geo.check(f, "f")
    _checked_spec(post, geo, "post", 0)
    _checked_spec(pre, geo, "pre")
    if gate_act not in ACTS:
        raise ValueError(f"gate_act must be one of {sorted(ACTS)}, got {gate_act!r}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    mode = 0
    if gate is not None:
        if gate.shape == x.shape and (gate.dtype == x.dtype or x.dim() > 2):      # [B, C] with another type: one for each of B
            geo.check(gate, "gate")
            mode = 3
        elif gate.shape in ((geo.C,), (geo.B, geo.C)):
            if gate.device != geo.device or not gate.is_floating_point():
                raise ValueError(f"gate: floating-point values on {geo.device} expected, got {gate.dtype} on {gate.device}")
            mode = 1 if gate.dim() == 1 else 2
            gate = gate.float().contiguous()
        else:
            raise ValueError(f"gate of shape {tuple(gate.shape)}: ({geo.C},), ({geo.B}, {geo.C}) or {tuple(x.shape)} expected")
    return _run(geo, x, f, gate, mode, ACTS[gate_act] if gate is not None else 0, float(scale), post, pre)


class ChannelNorm(nn.Module):
    """A norm over the channels with its parameters (fp32): ``weight`` and, for kind "layer" unless ``bias=False``, ``bias``."""

    def __init__(self, channels: int, kind: str = "rms", eps: float = 1e-6, bias: Optional[bool] = None, channel_dim: int = 1):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
        self.kind, self.eps, self.channel_dim = kind, eps, channel_dim
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if (kind == "layer" if bias is None else bias) else None

    @property
    def spec(self) -> NormSpec:
        return NormSpec(self.kind, self.weight, self.bias, self.eps)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return channel_norm(x, self.spec, self.channel_dim)


class GatedResidualStack(nn.Module):
    """Residual branches with a norm before and after each: ``x <- x + residual_scale * act(gate_i) * N_post_i(block_i(N_pre_i(x)))``.

    blocks: modules that keep their input's shape (``ResidualDenseBlock``, for instance).  gate: "channel" (a learned [C]
    per block, starting at ``gate_init``), "input" (``forward(x, gates)`` takes one per block, [B, C] or like x) or None.
    The end of each branch and the norm in front of the next one are one launch."""

    def __init__(self, blocks: Sequence[nn.Module], channels: int, kind: str = "rms", gate: Optional[str] = "channel",
                 gate_act: str = "none", gate_init: float = 1.0, residual_scale: float = 0.2, eps: float = 1e-6, channel_dim: int = 1):
        super().__init__()
        if gate not in ("channel", "input", None):
            raise ValueError(f"gate must be 'channel', 'input' or None, got {gate!r}")
        if gate_act not in ACTS:
            raise ValueError(f"gate_act must be one of {sorted(ACTS)}, got {gate_act!r}")
        self.blocks = nn.ModuleList(blocks)
        if not len(self.blocks):
            raise ValueError("no blocks")
        norms = lambda: nn.ModuleList(ChannelNorm(channels, kind, eps, channel_dim=channel_dim) for _ in self.blocks)  # noqa: E731
        self.pre, self.post = norms(), norms()
        self.gate, self.gate_act, self.residual_scale, self.channel_dim = gate, gate_act, residual_scale, channel_dim
        self.gates = nn.ParameterList(nn.Parameter(torch.full((channels,), float(gate_init))) for _ in self.blocks) \
            if gate == "channel" else None

    def forward(self, x: torch.Tensor, gates: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
        if (gates is not None) != (self.gate == "input") or (gates is not None and len(gates) != len(self.blocks)):
            raise ValueError(f"gates: {'one for each of the ' + str(len(self.blocks)) + ' blocks' if self.gate == 'input' else 'none'} expected")
        gates = list(gates) if gates is not None else list(self.gates) if self.gates is not None else [None] * len(self.blocks)
        h = self.pre[0](x)
        for i, block in enumerate(self.blocks):
            last = i + 1 == len(self.blocks)
            x = gated_residual(x, block(h), post=self.post[i].spec, gate=gates[i], gate_act=self.gate_act, scale=self.residual_scale,
                               pre=None if last else self.pre[i + 1].spec, channel_dim=self.channel_dim)
            if not last:
                x, h = x
        return x
