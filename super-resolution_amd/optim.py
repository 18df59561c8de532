"""AdamW over a list of tensors (``srx_adamw_step``): what ``train.FlatAdam`` does not cover.

``FlatAdam`` is ``torch.optim.Adam`` (esrgan/train_esrgan.py:134-135) over ONE flat fp32 range.  ``AdamW`` takes the
parameters as they are — any number of tensors, in groups with a learning rate and a (decoupled) weight decay of
their own, fp32 or bf16 with an fp32 master — and adds clipping by the global gradient norm, the skip of a step
whose gradients are not finite, and moments in 8 bits (2 bytes and a bit per parameter instead of 8).  All
decisions are taken on the device: a step never waits for the host and can be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes as C
import math
import warnings
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from . import _lib as L
from . import engine

_ptr = torch.Tensor.data_ptr
_MOVED, _ODD, _BF16 = 1, 2, 4              # flags of the host module's gather()
_DTYPE_ID = {torch.bfloat16: L.BF16, torch.float32: L.F32}


def _in_memory(t: torch.Tensor, what: str) -> torch.Tensor:
    """t with its values in memory: a negative view and a tensor of zeros without memory are copied (both count as contiguous)."""
    if t._is_zerotensor():
        return t.detach().clone()
    if L.host().unheld([t]) >= 0:          # a storage can be resized under its tensors
        raise ValueError(f"{what}: its memory has been freed")
    return t.detach().clone() if t.is_neg() else t


def decay_groups(module: torch.nn.Module, weight_decay: float = 1e-2) -> List[dict]:
    """Two parameter groups of a module, in ``parameters()`` order within each: tensors with two or more dimensions
    (kernels) decay; norm weights, gates and biases do not."""
    params = [p for p in module.parameters() if p.requires_grad]
    groups = [{"params": [p for p in params if p.dim() >= 2], "weight_decay": weight_decay},
              {"params": [p for p in params if p.dim() < 2], "weight_decay": 0.0}]
    return [g for g in groups if g["params"]]


class AdamW:
    """One step = ``p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)`` (``torch.optim.AdamW``).

    params: tensors, or dicts ``{"params": [...], "lr": ..., "betas": ..., "eps": ..., "weight_decay": ...}`` (at most 32);
        contiguous fp32 or bf16 tensors on one GPU.  A bf16 parameter gets an fp32 master copy; writing the
        parameter (loading a checkpoint, say) also moves its master.
    state_bits: 32, or 8: moments of one byte with a scale for every 256 elements of a tensor.
    rounding: of 8-bit moments.  "random" keeps their averages (with the same bits for the same inputs): the choice for
        training.  "nearest", the default, gives the nearest codes, but its second moments do not follow a slow average: with
        beta2 = 0.999 a value's ratio to the largest of its 256 stays put until one gradient's square exceeds 30 to 60 times
        it.  A warning says so where neither is given.
    max_grad_norm: gradients are scaled by ``min(1, max_grad_norm / (norm + 1e-6))``, norm over all tensors.
    skip_nonfinite: a step whose gradient norm is infinite or NaN changes nothing.

    ``param_groups`` holds the hyper-parameters under torch's names and is read at every step; ``lr`` sets one learning
    rate for all, ``schedule_lr`` one that respects the groups' own.
    A captured step replays with the hyper-parameters and ``grad_scale`` it was captured with, and reads its gradients
    where they were then; its step count advances.  Where parameters have got new storage since, one eager step
    makes it follow them.  One optimizer's steps share its state and workspaces: they must not overlap.  To autograd a step is an
    in-place change of every parameter that it moves: a graph that saved one of them refuses its backward pass."""

    def __init__(self, params: Iterable, lr: float = 2e-4, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, max_grad_norm: Optional[float] = None,
                 skip_nonfinite: bool = False, rounding: Optional[str] = None):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if rounding not in (None, "nearest", "random"):
            raise ValueError(f"rounding must be 'nearest' or 'random', got {rounding!r}")
        if rounding == "random" and state_bits == 32:
            raise ValueError("rounding: 32-bit moments are not rounded")
        if max_grad_norm is not None and not 0 < max_grad_norm < math.inf:
            raise ValueError(f"max_grad_norm must be positive and finite, got {max_grad_norm}")
        params = list(params)
        if not params:
            raise ValueError("no parameters")
        if not all(isinstance(g, dict) for g in params):
            if any(isinstance(g, dict) for g in params):
                raise TypeError("params: tensors or dicts, not both")
            params = [{"params": params}]
        if len(params) > L.ADAMW_MAX_GROUPS:
            raise ValueError(f"{len(params)} parameter groups: at most {L.ADAMW_MAX_GROUPS} are supported")
        defaults = {"lr": lr, "betas": tuple(betas), "eps": eps, "weight_decay": weight_decay}
        self.param_groups: List[dict] = []
        for g in params:
            if not set(g) <= {"params", "lr", "betas", "eps", "weight_decay", "initial_lr"}:
                raise ValueError(f"unknown keys in a parameter group: {sorted(set(g) - set(defaults) - {'params'})}")
            ps = g["params"]
            ps = [ps] if isinstance(ps, torch.Tensor) else list(ps)
            group = {**defaults, **g, "params": ps}
            group["betas"] = tuple(group["betas"])
            group.setdefault("initial_lr", group["lr"])
            self.param_groups.append(group)
        self._lr_ratio = [g["lr"] / lr if lr > 0 else 1.0 for g in self.param_groups]
        self.params: List[torch.Tensor] = [p for g in self.param_groups for p in g["params"]]
        if not self.params:
            raise ValueError("no parameters")
        for i, p in enumerate(self.params):
            if not isinstance(p, torch.Tensor):
                raise TypeError(f"parameter {i} is a {type(p).__name__}, not a tensor")
            if p.device.type != "cuda":
                raise RuntimeError(f"libsrx runs on a ROCm GPU only (parameter {i} is on {p.device})")
            if p.device != self.params[0].device:
                raise ValueError(f"parameters on {self.params[0].device} and on {p.device}: all must be on one GPU")
            if p.dtype not in _DTYPE_ID:
                raise ValueError(f"parameter {i} is {p.dtype}: float32 or bfloat16 are supported")
        self._check_hyper()
        if state_bits == 8 and rounding is None:
            warnings.warn("AdamW: 8-bit moments rounded to nearest do not follow their average over many steps; give rounding='random' for "
                          "training (or 'nearest' for this rounding without a warning)", stacklevel=2)
        self.device = self.params[0].device
        self.state_bits, self.max_grad_norm, self.skip_nonfinite = state_bits, max_grad_norm, bool(skip_nonfinite)
        self.rounding = rounding or "nearest"
        self._lib = L.lib()
        self._n = [p.numel() for p in self.params]
        self._shapes = [p.shape for p in self.params]
        self._dtypes = [p.dtype for p in self.params]
        blocks = [-(-n // L.ADAMW_BLOCK) for n in self._n]
        self._first = [0]
        for b in blocks:
            self._first.append(self._first[-1] + b)
        self.nblocks = self._first[-1]
        chunks = [-(-n // L.ADAMW_CHUNK) for n in self._n]
        start = np.concatenate([[0], np.cumsum(chunks)]).astype(np.int32)
        table = np.empty((int(start[-1]), 2), dtype=np.int32)
        table[:, 0] = np.repeat(np.arange(len(chunks)), chunks)
        table[:, 1] = np.arange(start[-1]) - np.repeat(start[:-1], chunks)
        dev, padded = self.device, L.ADAMW_BLOCK * self.nblocks
        with torch.cuda.device(dev):
            zeros = lambda n, t=torch.float32: torch.zeros(max(n, 1), dtype=t, device=dev)  # noqa: E731
            self._chunks = torch.from_numpy(table.reshape(-1) if table.size else np.zeros(2, np.int32)).to(dev)
            self._m = torch.zeros(padded, dtype=torch.float32 if state_bits == 32 else torch.uint8, device=dev)
            self._v = torch.zeros_like(self._m)
            self._m_scale, self._v_scale = (zeros(self.nblocks), zeros(self.nblocks)) if state_bits == 8 else (None, None)
            self._steps = zeros(len(self.params), torch.int32)
            self._coef = zeros(4 + 10 * len(self.params))
            self._partial = zeros(int(start[-1]), torch.float64)
            half = [n if t == torch.bfloat16 else 0 for n, t in zip(self._n, self._dtypes)]
            self._master_at = [0]
            for n in half:
                self._master_at.append(self._master_at[-1] + n)
            #: fp32 masters of the bf16 parameters, one after the other (None: there are none)
            self.master = zeros(self._master_at[-1]) if sum(half) else None
            self._tensors: Optional[torch.Tensor] = None
            self._bind()
            self._addresses, self._types = np.zeros(len(self.params), np.uint64), np.zeros(len(self.params), np.uint8)
            self._addresses_at, self._types_at = self._addresses.ctypes.data, self._types.ctypes.data
            self._gather, self._written, self._none = L.host().gather, L.host().written, [None] * len(self.params)
            self._own = [t for t in (self._m, self._v, self.master) if t is not None]
            self._copy_masters()
            d = self._desc = L.AdamwDesc()
            d.state_bits, d.ntensors, d.ngroups = state_bits, len(self.params), len(self.param_groups)
            d.rounding = rounding == "random"
            self._start = start
            d.chunks, d.chunk_start = self._chunks.data_ptr(), start.ctypes.data
            d.m, d.v = self._m.data_ptr() or self._steps.data_ptr(), self._v.data_ptr() or self._steps.data_ptr()
            if state_bits == 8:
                d.m_scale, d.v_scale = self._m_scale.data_ptr(), self._v_scale.data_ptr()
            d.steps, d.coef, d.partial = self._steps.data_ptr(), self._coef.data_ptr(), self._partial.data_ptr()
            self._groups = (L.AdamwGroup * len(self.param_groups))()
            d.groups = C.addressof(self._groups)
            torch.cuda.current_stream(dev).synchronize()     # ready for a first step on any stream

    # ---------------------------------------------------------------- hyper-parameters
    @property
    def lr(self) -> float:
        return self.param_groups[0]["lr"]

    @lr.setter
    def lr(self, value: float) -> None:
        for g in self.param_groups:
            g["lr"] = value

    def schedule_lr(self, value: float) -> None:
        """The learning rate of a schedule: a group that was given one of its own keeps its ratio to the constructor's ``lr``."""
        for g, ratio in zip(self.param_groups, self._lr_ratio):
            g["lr"] = value * ratio

    def _check_hyper(self, groups: Optional[List[dict]] = None) -> None:
        for i, g in enumerate(self.param_groups if groups is None else groups):
            b = g["betas"]
            if not (0 <= g["lr"] < math.inf and len(b) == 2 and 0 <= b[0] < 1 and 0 <= b[1] < 1 and 0 <= g["eps"] < math.inf
                    and 0 <= g["weight_decay"] < math.inf):
                raise ValueError(f"parameter group {i}: lr, eps and weight_decay must be finite and not negative, betas in [0, 1): "
                                 f"{ {k: v for k, v in g.items() if k != 'params'} }")

    # ---------------------------------------------------------------- tables
    def _bind(self) -> None:
        """Write the parameters' addresses into the device table: at construction, and again when a parameter has got new
        storage since (``module.to()``, ``flatten_parameters``)."""
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: the parameters have got new storage; run one step outside of the capture first")
        ptrs = list(map(_ptr, self.params))
        for i, p in enumerate(self.params):
            if p.device != self.device or p.dtype != self._dtypes[i] or p.numel() != self._n[i]:
                raise RuntimeError(f"AdamW: parameter {i} was {self._dtypes[i]} of {self._n[i]} elements on {self.device} and is now "
                                   f"{p.dtype} of {p.numel()} on {p.device}: build a new optimizer")
            if not p.is_contiguous():
                raise ValueError(f"AdamW: parameter {i} is not contiguous")
            if p.is_neg():
                raise ValueError(f"AdamW: parameter {i} is a negative view: its memory holds other values than it")
        freed = L.host().unheld(self.params)
        if freed >= 0:
            raise ValueError(f"AdamW: the memory of parameter {freed} has been freed")
        spans = sorted((a, a + n * p.element_size(), i) for i, (a, n, p) in enumerate(zip(ptrs, self._n, self.params)) if n)
        for (_, end, i), (begin, _, k) in zip(spans, spans[1:]):
            if begin < end:
                raise ValueError(f"AdamW: parameters {i} and {k} share memory (or are the same tensor)")
        if len({id(p) for p in self.params}) != len(self.params):
            raise ValueError("AdamW: a parameter is given twice")
        # views of one buffer that cover it without gaps: their gradients may come as one buffer too
        base, esize = (spans[0][0], self.params[0].element_size()) if spans else (0, 1)
        self._flat = bool(spans) and len(set(self._dtypes)) == 1 and spans[-1][1] - base == sum(self._n) * esize
        arr = (L.AdamwTensor * len(self.params))()
        i = 0
        for gi, g in enumerate(self.param_groups):
            for _ in g["params"]:
                t = arr[i]
                t.p, t.n, t.first_block, t.group = ptrs[i] or None, self._n[i], self._first[i], gi
                if self._dtypes[i] == torch.bfloat16:
                    t.master = self.master.data_ptr() + 4 * self._master_at[i]
                t.g_off = (ptrs[i] - base) // esize if self._flat and self._n[i] else 0
                i += 1
        raw = torch.frombuffer(bytearray(C.string_at(C.addressof(arr), C.sizeof(arr))), dtype=torch.uint8)
        if self._tensors is None:
            self._tensors = raw.to(self.device)
        else:
            # in place: a captured step holds the table's address, and follows the parameters too
            torch.cuda.synchronize(self.device)      # steps in flight still read the old entries
            self._tensors.copy_(raw)
        self._bound = np.array(ptrs + [2 * n + (t == torch.bfloat16) for n, t in zip(self._n, self._dtypes)], dtype=np.uint64)

    def _copy_masters(self) -> None:
        for i, p in enumerate(self.params):
            if p.dtype == torch.bfloat16:
                self.master[self._master_at[i]:self._master_at[i + 1]].copy_(p.detach().reshape(-1))

    # ---------------------------------------------------------------- the step
    def step(self, grads: Union[None, torch.Tensor, Sequence[Optional[torch.Tensor]]] = None,
             grad_scale: float = 1.0) -> Optional[torch.Tensor]:
        """One step on the current stream.  grads: None (each parameter's ``.grad``), a list with one gradient (fp32 or
        bf16) or None per parameter — None leaves that parameter, its moments and its step count as they are — or,
        where the parameters are views that cover one flat buffer, one flat gradient of the same layout.
        ``grad_scale`` multiplies every gradient first (1 / loss scale).  Returns the gradient norm before clipping
        (0-dim tensor, not synchronised) if ``max_grad_norm`` or ``skip_nonfinite`` is set, else None."""
        if torch._C._cuda_getDevice() != self.device.index:
            with torch.cuda.device(self.device):
                return self.step(grads, grad_scale)
        if not math.isfinite(grad_scale):
            raise ValueError(f"grad_scale must be finite, got {grad_scale}")
        d = self._desc
        if isinstance(grads, torch.Tensor):
            if self._gather(self.params, self._none, self._bound, self._addresses, self._types, self.device.index) & _MOVED:
                self._bind()
            if not self._flat:
                raise ValueError("a flat gradient needs parameters of one type that are views covering one flat buffer")
            if grads.device != self.device or grads.dtype not in _DTYPE_ID or grads.numel() != sum(self._n) or not grads.is_contiguous():
                raise ValueError(f"flat gradient: {sum(self._n)} contiguous float32 or bfloat16 values on {self.device} expected, got "
                                 f"{grads.dtype} of {tuple(grads.shape)} on {grads.device}")
            grads = _in_memory(grads, "flat gradient")
            d.grads, d.grad_dtypes = None, None
            d.flat_grad, d.flat_dtype = grads.data_ptr(), _DTYPE_ID[grads.dtype]
            if grads.numel() == 0:
                return self._empty_norm()
        else:
            # one pass over both lists: addresses, types, and whether anything is not as it should be
            if grads is not None and type(grads) is not list:
                grads = list(grads)
            index = self.device.index
            flags = self._gather(self.params, grads, self._bound, self._addresses, self._types, index)
            if flags & _MOVED:
                self._bind()
            if flags & _ODD:
                grads = self._taken(grads)
                flags = self._gather(self.params, grads, self._bound, self._addresses, self._types, index)
            d.grads, d.flat_grad = self._addresses_at, None
            d.grad_dtypes = self._types_at if flags & _BF16 else None
        self._check_hyper()
        for q, g in zip(self._groups, self.param_groups):
            q.lr, (q.beta1, q.beta2), q.eps, q.weight_decay = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        d.tensors = self._tensors.data_ptr()
        d.grad_scale, d.max_norm, d.skip_nonfinite = grad_scale, self.max_grad_norm or 0.0, self.skip_nonfinite
        norm = None
        if self.max_grad_norm or self.skip_nonfinite:
            norm = torch.empty((), dtype=torch.float32, device=self.device)
            d.norm = norm.data_ptr()
        L.check(self._lib.srx_adamw_step(C.byref(d), torch._C._cuda_getCurrentRawStream(self.device.index)), "srx_adamw_step")
        self._written(self.params, None if d.flat_grad else self._addresses, self._own)
        return norm

    def _empty_norm(self):
        return torch.zeros((), device=self.device) if self.max_grad_norm or self.skip_nonfinite else None

    def _taken(self, grads) -> list:
        """Gradients that gather() cannot take as they are: brought into order, or refused."""
        grads = [p.grad for p in self.params] if grads is None else grads
        for i, (g, p) in enumerate(zip(grads, self.params)):
            if g is None:
                continue
            if g.shape != p.shape or g.device != p.device:
                raise ValueError(f"gradient {i} has shape {tuple(g.shape)} on {g.device}, its parameter {tuple(p.shape)} on {p.device}")
            if g.dtype not in _DTYPE_ID or g.layout != torch.strided:
                raise ValueError(f"gradient {i}: a dense float32 or bfloat16 tensor expected, got {g.dtype}, {g.layout}")
        return [g if g is None else _in_memory(g, f"gradient {i}").contiguous() for i, g in enumerate(grads)]

    def zero_grad(self, set_to_none: bool = True) -> None:
        for p in self.params:
            if p.grad is not None:
                if set_to_none:
                    p.grad = None
                else:
                    p.grad.zero_()

    # ---------------------------------------------------------------- state
    def moments(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) in fp32, flat: every parameter's start at a multiple of 256 elements, zeros between.  The optimizer's own
        buffers with 32-bit moments; with 8-bit ones new tensors of the values that they stand for."""
        if self.state_bits == 32:
            return self._m, self._v
        with torch.cuda.device(self.device):
            m, v = (torch.empty(self._m.numel(), dtype=torch.float32, device=self.device) for _ in range(2))
            L.check(self._lib.srx_adamw_moments_from8(self._m.data_ptr(), self._v.data_ptr(), self._m_scale.data_ptr(),
                                                      self._v_scale.data_ptr(), m.data_ptr(), v.data_ptr(), self.nblocks,
                                                      engine.stream_ptr(self.device)), "srx_adamw_moments_from8")
        return m, v

    def load_moments(self, m: torch.Tensor, v: torch.Tensor, step: Union[int, Sequence[int]],
                     master: Optional[torch.Tensor] = None) -> None:
        """Set the whole state: moments as :meth:`moments` returns them, step counts (one, or one per parameter), and the
        masters of the bf16 parameters (None: taken from the parameters)."""
        steps = [int(step)] * len(self.params) if isinstance(step, int) else [int(k) for k in step]
        if len(steps) != len(self.params) or not 0 <= min(steps) <= max(steps) < 2 ** 31:
            raise ValueError("step: one count from 0 to 2^31 - 1, or one per parameter")
        for name, t, n in (("m", m, self._m.numel()), ("v", v, self._v.numel())) + \
                ((("master", master, self._master_at[-1]),) if master is not None else ()):
            if t.numel() != n or t.dtype != torch.float32 or t.device != self.device:
                raise ValueError(f"{name}: {n} float32 values on {self.device} expected, got {t.dtype} of {t.numel()} on {t.device}")
        with torch.cuda.device(self.device), torch.no_grad():
            if self.state_bits == 32:
                self._m.copy_(m.reshape(-1))
                self._v.copy_(v.reshape(-1))
            else:
                m, v = (t.detach().reshape(-1).clone() for t in (m, v))       # contiguous and aligned
                L.check(self._lib.srx_adamw_moments_to8(m.data_ptr(), v.data_ptr(), self._m.data_ptr(), self._v.data_ptr(),
                                                        self._m_scale.data_ptr(), self._v_scale.data_ptr(), self.nblocks,
                                                        engine.stream_ptr(self.device)), "srx_adamw_moments_to8")
            self._steps.copy_(torch.tensor(steps, dtype=torch.int32))
            if self.master is not None:
                if master is None:
                    self._copy_masters()
                else:
                    self.master.copy_(master.reshape(-1))
            torch.cuda.current_stream(self.device).synchronize()

    @property
    def step_counts(self) -> List[int]:
        """Steps taken by each parameter (reads the device)."""
        return self._steps[:len(self.params)].tolist()

    def state_dict(self) -> dict:
        """The ``torch.optim.AdamW.state_dict()`` layout with fp32 moments whatever ``state_bits`` (they load back to the
        same 8 bits); a bf16 parameter's state also holds its ``master``."""
        m, v = self.moments()
        state = {}
        for i, (n, shp, t) in enumerate(zip(self._n, self._shapes, self.step_counts)):
            if t == 0 and self.master is None:
                continue
            at = L.ADAMW_BLOCK * self._first[i]
            state[i] = {"step": torch.tensor(float(t)), "exp_avg": m[at:at + n].view(shp).clone(),
                        "exp_avg_sq": v[at:at + n].view(shp).clone()}
            if self._dtypes[i] == torch.bfloat16:
                state[i]["master"] = self.master[self._master_at[i]:self._master_at[i + 1]].view(shp).clone()
        groups, k = [], 0
        for g in self.param_groups:
            groups.append({**{key: g[key] for key in ("lr", "initial_lr", "betas", "eps", "weight_decay")},
                           "amsgrad": False, "maximize": False, "foreach": None, "capturable": False, "differentiable": False,
                           "fused": None, "decoupled_weight_decay": True, "params": list(range(k, k + len(g["params"])))})
            k += len(g["params"])
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, sd: dict) -> None:
        """Accepts a state_dict written by this class (any ``state_bits``) or by ``torch.optim.AdamW`` over the same parameters
        in the same groups.  One that is refused changes nothing."""
        groups = sd["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError(f"optimizer state_dict does not match: groups of {[len(g['params']) for g in groups]} parameters, "
                             f"{[len(g['params']) for g in self.param_groups]} here")
        if any(g.get("amsgrad") or g.get("maximize") for g in groups):
            raise ValueError("optimizer state_dict with amsgrad or maximize: neither is supported")
        order = [k for g in groups for k in g["params"]]
        m = torch.zeros(self._m.numel(), dtype=torch.float32, device=self.device)
        v, steps = torch.zeros_like(m), []
        master = None
        if self.master is not None:
            master = torch.cat([p.detach().reshape(-1).float() for p in self.params if p.dtype == torch.bfloat16])
        for i, (k, n, shp) in enumerate(zip(order, self._n, self._shapes)):
            st = sd["state"].get(k)
            steps.append(int(float(st["step"])) if st is not None else 0)
            if st is None:
                continue
            for key in ("exp_avg", "exp_avg_sq", "master"):
                if key in st and tuple(st[key].shape) != tuple(shp):
                    raise ValueError(f"optimizer state for parameter {i}: {key} has shape {tuple(st[key].shape)}, expected {tuple(shp)}")
            at = L.ADAMW_BLOCK * self._first[i]
            m[at:at + n].copy_(st["exp_avg"].reshape(-1))
            v[at:at + n].copy_(st["exp_avg_sq"].reshape(-1))
            if "master" in st and self._dtypes[i] == torch.bfloat16:
                master[self._master_at[i]:self._master_at[i + 1]].copy_(st["master"].reshape(-1))
        hyper = [{**{key: float(new[key]) for key in ("lr", "eps", "weight_decay")}, "betas": tuple(new["betas"]),
                  "initial_lr": new.get("initial_lr", g["initial_lr"])} for g, new in zip(self.param_groups, groups)]
        self._check_hyper(hyper)
        self.load_moments(m, v, steps, master)
        for g, new in zip(self.param_groups, hyper):
            g.update(new)
