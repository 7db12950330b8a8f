"""`IrrepsNorm` and `GatedResidual`: what stands in front of and behind an equivariant block of a network.

No counterpart in the reference.  Features are rows of irrep blocks (mul channels x dim components); per row and block
``r(t) = (mean of t^2 over the block's channels and components + eps)^-1/2``:

* ``IrrepsNorm``: ``y = w x r(x)``, one weight per channel;
* ``GatedResidual``: ``h = x + s act(g) y r(y)`` for the block's output ``y``, one gate per row and channel, one scale per channel;
  with ``norm_output`` also ``n = w h r(h)``, the norm in front of the next block, in the same pass.

A block's components share their factors, so both are equivariant, and so are their gradients with activations kept in full.  With
``saved_activations="int8"`` the forward results still are; the gradients are not: the step of a block follows its largest component, which a
rotation changes, so a gradient is off by up to 1/127 in a direction that depends on the frame.  Forces from such gradients are neither covariant nor
exactly a derivative of the energy.

The kernels are ``csrc/norm_kernels.cuh``.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib, profiling
from ..executor import dtype_code
from ..irreps import Irreps, IrrepsLayout

_NAMES = {_lib.NORM_BRANCH: "gated_residual_", _lib.NORM_ALONE: "irreps_norm_", _lib.NORM_BOTH: "gated_residual_norm_"}
SAVED_ACTIVATIONS = ("full", "int8")
_TYPES = (torch.float32, torch.float64, torch.bfloat16, torch.float16)
_ROUNDED = (torch.bfloat16, torch.float16)


def check_saved_activations(value: str) -> bool:
    """True for ``"int8"``."""
    if value not in SAVED_ACTIVATIONS:
        raise ValueError(f"saved_activations must be one of {SAVED_ACTIVATIONS}, got {value!r}")
    return value == "int8"


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride along the row and rows that do not overlap (or are all the same one)."""
    if t.is_contiguous() or (t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.stride(0) == 0 or t.shape[0] <= 1):
        return t
    return t.contiguous()


def _features(like: torch.Tensor, width: int) -> torch.Tensor:
    """Dense rows of ``width`` values for the rows of ``like``."""
    return torch.empty_like(like) if like.shape[1] == width and like.is_contiguous() else like.new_empty((like.shape[0], width))


class _Block:
    """What the modules share: the irreps' blocks, the layout and the launches."""

    def __init__(self, irreps: Irreps, layout: IrrepsLayout, eps: float, mode: int, gate: Optional[str], int8: bool):
        muls = [(mul, ir.dim) for mul, ir in irreps if mul > 0]
        if not 1 <= len(muls) <= _lib.NORM_MAX_BLOCKS:
            raise ValueError(f"irreps of 1 to {_lib.NORM_MAX_BLOCKS} blocks are supported, got {irreps}")
        if not 0 < eps < float("inf"):
            raise ValueError(f"eps must be positive and finite, got {eps}")
        self.blocks = (_lib.NormBlock * len(muls))(*muls)
        self.dim, self.channels = sum(m * d for m, d in muls), sum(m for m, _ in muls)
        self.layout, self.eps, self.mode, self.gate, self.int8 = layout, eps, mode, gate, int8
        pad = lambda n: (n + 15) // 16 * 16  # noqa: E731
        features = sum(pad(m * d) for m, d in muls)
        self.code_bytes = features * (2 if mode == _lib.NORM_BOTH else 1) + (sum(pad(m) for m, _ in muls) if gate else 0)
        self._arguments = {}
        self.stats_stride = 8 if int8 and mode == _lib.NORM_BOTH else 4

    def __getstate__(self):
        state = dict(self.__dict__)
        state["blocks"], state["_arguments"] = [(b.mul, b.dim) for b in self.blocks], {}
        return state

    def __setstate__(self, state):
        self.__dict__.update(state)
        self.blocks = (_lib.NormBlock * len(state["blocks"]))(*state["blocks"])

    def check(self, name: str, t: torch.Tensor, width: int, like: Optional[torch.Tensor] = None) -> None:
        shape = t.shape
        if len(shape) != 2 or shape[1] != width:
            raise ValueError(f"{name} must have shape (batch, {width}), got {tuple(shape)}")
        if not t.is_cuda:
            raise RuntimeError("cuequivariance_b200 executes on CUDA devices only (there is no CPU fallback)")
        if like is not None and (shape[0] != like.shape[0] or t.dtype != like.dtype or t.device != like.device):
            raise ValueError(f"{name} must have the rows, dtype and device of x: {tuple(shape)} {t.dtype} {t.device} "
                             f"against {tuple(like.shape)} {like.dtype} {like.device}")

    def check_x(self, x: torch.Tensor) -> None:
        self.check("x", x, self.dim)
        if x.dtype not in _TYPES:
            raise ValueError(f"unsupported dtype {x.dtype}")
        if self.int8 and x.dtype == torch.float64:
            raise ValueError("saved_activations='int8' is for float32, bfloat16 and float16; float64 activations are kept in full")

    def check_parameter(self, name: str, t: Optional[torch.Tensor], x: torch.Tensor) -> None:
        if t is None:
            raise ValueError(f"{name} should not be None")
        if t.shape != (self.channels,) or t.device != x.device:
            raise ValueError(f"{name} must have shape ({self.channels},) on {x.device}, got {tuple(t.shape)} on {t.device}")
        if t.dtype not in _TYPES or (x.dtype == torch.float64) != (t.dtype == torch.float64):
            raise ValueError(f"{name} has dtype {t.dtype}, features {x.dtype}: float64 goes with float64 only")

    def arguments(self, mode: int, x: torch.Tensor, parameter: torch.Tensor) -> "_lib.NormArgs":
        """The argument block of a call, without pointers to tensors; what does not change from call to call is kept per type."""
        key = (mode, x.dtype, parameter.dtype, x.device)
        kept = self._arguments.get(key)
        if kept is None:
            a = _lib.NormArgs()
            a.struct_bytes, a.mode, a.gate, a.mul_ir = C.sizeof(a), mode, _lib.NORM_GATES[self.gate], int(self.layout is IrrepsLayout.mul_ir)
            a.dtype, a.param_dtype, a.num_blocks, a.stats_stride = dtype_code(x.dtype), dtype_code(parameter.dtype), len(self.blocks), self.stats_stride
            a.blocks, a.eps = self.blocks, self.eps
            a.status = _lib.status_word(x.device).data_ptr()
            kept = self._arguments[key] = bytes(a)
        a = _lib.NormArgs.from_buffer_copy(kept)
        a.rows = x.shape[0]
        return a

    def launch(self, which: str, a: "_lib.NormArgs", device: torch.device) -> None:
        L = _lib.lib()
        fn = L.cueq_b200_norm_forward if which == "forward" else L.cueq_b200_norm_backward
        with _lib.on_device(device), profiling.kernel(_NAMES[a.mode] + which):
            _lib.check(fn(C.byref(a), torch._C._cuda_getCurrentRawStream(device.index)))

    def forward(self, keep: bool, x, y, g, s, w):
        """(out, norm, codes, stats) - the last two for a backward pass to come."""
        x, y, g, s, w = (_rows(x), None if y is None else _rows(y), None if g is None else _rows(g),
                         None if s is None else s.contiguous(), None if w is None else w.contiguous())
        a = self.arguments(self.mode, x, s if s is not None else w)
        a.x, a.ldx = x.data_ptr(), x.stride(0)
        out = norm = codes = stats = None
        if y is not None:
            out = _features(x, self.dim)
            a.y, a.ldy, a.scale, a.out = y.data_ptr(), y.stride(0), s.data_ptr(), out.data_ptr()
        if g is not None:
            a.g, a.ldg = g.data_ptr(), g.stride(0)
        if w is not None:
            norm = _features(x, self.dim)
            a.weight, a.norm = w.data_ptr(), norm.data_ptr()
        if keep:
            stats = x.new_empty((x.shape[0], len(self.blocks), self.stats_stride), dtype=torch.float64 if x.dtype == torch.float64 else torch.float32)
            a.stats = stats.data_ptr()
            if self.int8:
                codes = x.new_empty((x.shape[0], self.code_bytes), dtype=torch.int8)
                a.codes, a.ld_codes = codes.data_ptr(), self.code_bytes
        if x.shape[0]:
            self.launch("forward", a, x.device)
        return out, norm, codes, stats

    def kept(self, x, y, g, out, codes):
        """(y, g, h) for the backward pass, None where they are in codes or not read.  ``h``: what was normalised; behind a branch in 16
        bits, where the result has been rounded, x, from which the kernel forms it again."""
        if codes is not None:
            return None, None, None
        if self.mode == _lib.NORM_BOTH:
            return y, g, x if x.dtype in _ROUNDED else out
        return y, g, x if self.mode == _lib.NORM_ALONE else None

    def backward(self, go, gn, y, g, h, codes, stats, s, w, need_s, need_w):
        """(dx, dy, dg, ds, dw); ``y``, ``g``, ``h`` as ``kept`` returned them; ds, dw None where they are not needed."""
        mode = self.mode if gn is not None else _lib.NORM_BRANCH      # a norm without a cotangent does not count
        like = gn if gn is not None else go
        s, w = (None if t is None else t.contiguous() for t in (s, w))
        a = self.arguments(mode, like, s if s is not None else w)
        rows, dx, dy, dg, ds, dw = like.shape[0], go, None, None, None, None
        # copies of operands live until the launch
        go, gn, y, g, h = (None if t is None else _rows(t) for t in (go, gn, y, g, h))
        if go is not None:
            a.go, a.ldgo = go.data_ptr(), go.stride(0)
        if mode & _lib.NORM_BRANCH:
            dy = _features(like, self.dim)
            a.scale, a.dy = s.data_ptr(), dy.data_ptr()
            if need_s:
                ds = torch.empty_like(s)
                a.dscale = ds.data_ptr()
            if y is not None:
                a.y, a.ldy = y.data_ptr(), y.stride(0)
            if self.gate:
                dg = _features(like, self.channels)
                a.dg = dg.data_ptr()
                if g is not None:
                    a.g, a.ldg = g.data_ptr(), g.stride(0)
        if mode & _lib.NORM_ALONE:
            a.gn, a.ldgn = gn.data_ptr(), gn.stride(0)
            dx = _features(like, self.dim)
            a.weight, a.dx = w.data_ptr(), dx.data_ptr()
            if need_w:
                dw = torch.empty_like(w)
                a.dweight = dw.data_ptr()
            if h is not None:
                a.h, a.ldh = a.x, a.ldx = h.data_ptr(), h.stride(0)
        a.stats = stats.data_ptr()
        if codes is not None:
            a.codes, a.ld_codes = codes.data_ptr(), self.code_bytes
        if rows:
            a.parts_values = -1
            if ds is not None or dw is not None:
                n = max(_lib.lib().cueq_b200_norm_parts(C.byref(a)), 0)
                parts = stats.new_empty(n)
                a.parts, a.parts_values = parts.data_ptr(), n
            self.launch("backward", a, like.device)
        else:
            ds, dw = (None if t is None else t.zero_() for t in (ds, dw))
        return dx, dy, dg, ds, dw


class _Norm(torch.autograd.Function):
    """One pass over the rows each way.  Kept for the backward pass: the statistics and y, g, h (alone, or behind a branch in 16 bits:
    x) as they are, or their codes."""

    @staticmethod
    def forward(ctx, block, x, y, g, s, w):
        out, norm, codes, stats = block.forward(True, x, y, g, s, w)
        ctx.block = block
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(*block.kept(x, y, g, out, codes), codes, stats, s, w)
        return tuple(t for t in (out, norm) if t is not None)

    @staticmethod
    def backward(ctx, *grads):
        # once_differentiable is there for the error on a second derivative; it costs 4 us a call
        return _gradients_once(ctx, *grads) if torch.is_grad_enabled() else _gradients(ctx, *grads)


def _gradients(ctx, *grads):
    block = ctx.block
    go = grads[0] if block.mode & _lib.NORM_BRANCH else None
    gn = grads[-1] if block.mode & _lib.NORM_ALONE else None
    if go is None and gn is None:
        return (None,) * 6
    y, g, h, codes, stats, s, w = ctx.saved_tensors
    need = ctx.needs_input_grad[1:]
    grads = block.backward(go, gn, y, g, h, codes, stats, s, w, need[3], need[4])
    return (None, *(t if n else None for t, n in zip(grads, need)))


_gradients_once = torch.autograd.function.once_differentiable(_gradients)


def _run(block: _Block, x, y, g, s, w):
    if torch.is_grad_enabled():
        for t in (x, y, g, s, w):
            if t is not None and t.requires_grad:
                return _Norm.apply(block, x, y, g, s, w)
    if forward_ad._current_level >= 0:
        return _Norm.apply(block, x, y, g, s, w)          # raises if an operand has a tangent, which needs no requires_grad
    out, norm, _, _ = block.forward(False, x, y, g, s, w)
    return tuple(t for t in (out, norm) if t is not None)


def _parameter(module: torch.nn.Module, name: str, given: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    own = getattr(module, name)
    if own is not None and given is not None:
        raise ValueError(f"Internal weights are used, {name} should be None")
    return own if own is not None else given


class IrrepsNorm(torch.nn.Module):
    """``forward(x, weight=None)``: ``x`` ``[batch, irreps.dim]`` in float32, float64, bfloat16 or float16, each irrep block of a row
    divided by the root of its mean square (over channels and components, plus ``eps``) and multiplied by one weight per channel.

    ``weight``: ``[irreps.num_irreps]``, channels in the order of the blocks; the module's own parameter when ``internal_weights``
    (ones at first).  float64 features go with float64 weights; others with weights of any other type.  Arithmetic, statistics and
    sums are in 32 bits (64 for float64); results are rounded once; a block whose sum of squares leaves that range (values from 1e19 on
    in float32 and bfloat16) counts as infinitely long and becomes zeros.  Rows may lie further apart than their width.  A row of an irrep block
    has to fit into the shared memory of an SM: up to 14,000 channels of scalars or 3,600 of l = 3 in float32 with a gradient to come, half
    of that in float64; longer blocks raise in the forward pass.

    ``saved_activations="int8"`` (not for float64) keeps x in 8 bits for the backward pass, per row and irrep block with a step of a power of two (off by at most
    1/127 of the block's largest magnitude); the forward result does not change; the gradients are then not equivariant: not for forces.
    First derivatives only, and none in forward mode."""

    def __init__(self, irreps, *, layout=None, eps: float = 1e-5, internal_weights: bool = True, saved_activations: str = "full",
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None):
        super().__init__()
        self.irreps = irreps if isinstance(irreps, Irreps) else Irreps(irreps)
        self.layout, self.eps, self.saved_activations = IrrepsLayout.parse(layout), eps, saved_activations
        self._block = _Block(self.irreps, self.layout, eps, _lib.NORM_ALONE, None, check_saved_activations(saved_activations))
        self.weight = torch.nn.Parameter(torch.ones(self._block.channels, device=device, dtype=dtype)) if internal_weights else None

    def extra_repr(self) -> str:
        return f"{self.irreps}, layout={self.layout.name}, eps={self.eps}, saved_activations={self.saved_activations}"

    def forward(self, x: torch.Tensor, weight: Optional[torch.Tensor] = None) -> torch.Tensor:
        weight = _parameter(self, "weight", weight)
        self._block.check_x(x)
        self._block.check_parameter("weight", weight, x)
        return _run(self._block, x, None, None, None, weight)[0]


class GatedResidual(torch.nn.Module):
    """``forward(x, update, gates=None, scale=None, weight=None)``: ``x + scale * act(gates) * norm(update)``, and with ``norm_output`` the
    pair of this and its norm with ``weight``.

    ``x``, ``update``: ``[batch, irreps.dim]``; ``gates``: ``[batch, irreps.num_irreps]``, one per channel in the order of the blocks,
    required unless ``gate`` is None (``"sigmoid"``, ``"silu"``); ``scale``, ``weight``: ``[irreps.num_irreps]``, the module's own parameters when
    ``internal_weights`` (``initial_scale`` and ones at first).  Gates below -87 are closed: both activations are 0 there.  ``norm`` is ``IrrepsNorm`` without weights - ``scale`` is its weight.

    Blocks of up to 9,600 channels of scalars or 3,200 of l = 3 in float32, 5,700 or 1,700 with ``norm_output``, half of that in float64.  Types,
    rows, rounding and ``saved_activations`` as in ``IrrepsNorm``.  Kept for the gradient are ``update``, ``gates`` and with ``norm_output`` the result, but in
    16 bits ``x`` in its place (the result has been rounded); in 8 bits ``update``, ``gates`` and the result before it was rounded.
    One pass each way: with ``norm_output`` the sum is neither read again for its norm nor its two gradients added by another pass."""

    def __init__(self, irreps, *, layout=None, gate: Optional[str] = "sigmoid", norm_output: bool = False, eps: float = 1e-5,
                 initial_scale: float = 1.0, internal_weights: bool = True, saved_activations: str = "full",
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None):
        super().__init__()
        if gate not in _lib.NORM_GATES:
            raise ValueError(f"gate must be one of {tuple(_lib.NORM_GATES)}, got {gate!r}")
        self.irreps = irreps if isinstance(irreps, Irreps) else Irreps(irreps)
        self.layout, self.gate, self.norm_output, self.eps = IrrepsLayout.parse(layout), gate, norm_output, eps
        self.saved_activations = saved_activations
        self._block = _Block(self.irreps, self.layout, eps, _lib.NORM_BOTH if norm_output else _lib.NORM_BRANCH, gate,
                             check_saved_activations(saved_activations))
        n = self._block.channels
        self.scale = torch.nn.Parameter(torch.full((n,), initial_scale, device=device, dtype=dtype)) if internal_weights else None
        self.weight = torch.nn.Parameter(torch.ones(n, device=device, dtype=dtype)) if internal_weights and norm_output else None

    def extra_repr(self) -> str:
        return (f"{self.irreps}, layout={self.layout.name}, gate={self.gate}, norm_output={self.norm_output}, eps={self.eps}, "
                f"saved_activations={self.saved_activations}")

    def forward(self, x: torch.Tensor, update: torch.Tensor, gates: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                weight: Optional[torch.Tensor] = None):
        b = self._block
        scale, weight = _parameter(self, "scale", scale), _parameter(self, "weight", weight)
        b.check_x(x)
        b.check("update", update, b.dim, x)
        if (gates is None) != (self.gate is None):
            raise ValueError("gates should be provided" if self.gate else "gates should be None: the module has no gate")
        if gates is not None:
            b.check("gates", gates, b.channels, x)
        b.check_parameter("scale", scale, x)
        if self.norm_output:
            b.check_parameter("weight", weight, x)
            if weight.dtype != scale.dtype:
                raise ValueError(f"scale and weight must have one dtype, got {scale.dtype} and {weight.dtype}")
        elif weight is not None:
            raise ValueError("weight should be None: the module has no norm_output")
        out = _run(b, x, update, gates, scale, weight)
        return out if self.norm_output else out[0]
