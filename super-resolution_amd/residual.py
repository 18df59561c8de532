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

The calls are no torch operations: tracing them (``torch.jit.trace``, ``make_fx``) and forward-mode differentiation are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Sequence

import torch
from torch import nn

from . import _lib as L

KINDS = {"none": 0, "rms": 1, "layer": 2}
ACTS = {"none": 0, "sigmoid": 1}
_LARGEST = torch.finfo(torch.float32).max


class NormSpec(NamedTuple):
    """One norm over the channels: ``kind`` "rms" (z / sqrt(mean z^2 + eps)) or "layer" ((z - mean) / sqrt(var + eps)), times
    ``weight`` plus ``bias`` ([C] each, None: 1 and 0)."""
    kind: str
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-6


def _checked_spec(spec: NormSpec, what: str, least: int = 1) -> None:
    if KINDS.get(spec.kind, -1) < least:
        raise ValueError(f"{what}: kind must be one of {[k for k, v in KINDS.items() if v >= least]}, got {spec.kind!r}")
    if not 1e-37 <= spec.eps <= _LARGEST:
        raise ValueError(f"{what}: eps must be positive (at least 1e-37) and a float32, got {spec.eps}")


_NONE = NormSpec("none", None, None, 1.0)
_resnorm = None


def _run(x, f, gate, gate_act, scale, post, pre, channel_dim):
    # the rest of the checks, memory orders, outputs and the autograd node: csrc/host.cpp
    global _resnorm
    if _resnorm is None:
        _resnorm = L.host().resnorm
    return _resnorm(x, f, gate, post.weight, post.bias, pre.weight, pre.bias, KINDS[post.kind], KINDS[pre.kind], post.eps, pre.eps, gate_act,
                    scale, channel_dim)


def channel_norm(x: torch.Tensor, norm: NormSpec, channel_dim: int = 1) -> torch.Tensor:
    """The norm of every pixel (row) of x over its channels."""
    if norm is None:
        raise ValueError("norm: a NormSpec is needed")
    _checked_spec(norm, "norm")
    return _run(x, None, None, 0, 1.0, _NONE, norm, channel_dim)


def gated_residual(x: torch.Tensor, f: torch.Tensor, *, post: Optional[NormSpec] = None, gate: Optional[torch.Tensor] = None,
                   gate_act: str = "none", scale: float = 1.0, pre: Optional[NormSpec] = None, channel_dim: int = 1):
    """``y = x + scale * act(gate) * N_post(f)``; with ``pre`` also ``h = N_pre(y)``: returns y, or (y, h).

    x, f: same shape, type and device.  post: the norm after the branch (None: none; kind "none": only its weight and
    bias).  gate: None, [C], [B, C] (B = x.shape[0]: one gate for each image or sequence) or a tensor like f; gate_act
    "none" or "sigmoid".  pre: the norm in front of the next branch.  Differentiable once, in everything but scale and eps."""
    if f is None:
        raise TypeError("f must be a tensor")
    if post is not None:
        _checked_spec(post, "post", 0)
    if pre is not None:
        _checked_spec(pre, "pre")
    if gate_act not in ACTS:
        raise ValueError(f"gate_act must be one of {sorted(ACTS)}, got {gate_act!r}")
    if not abs(scale) <= _LARGEST:
        raise ValueError(f"scale must be a finite float32, got {scale}")
    return _run(x, f, gate, ACTS[gate_act], scale, _NONE if post is None else post, _NONE if pre is None else pre, channel_dim)


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
