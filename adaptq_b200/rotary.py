"""Rotary: rotary positions on CUDA tensors (include/adaptq_paged.h: adaptq_rotary_apply).

The same object rotates the queries and keys that a caller handles itself, and goes along with
PagedKVCache.append and .attend, which rotate on the way.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from . import _lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

try:  # the handle of the current stream without a Stream object around it: 2 us less per call
    current_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
    def current_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def _has_tangent(x):
    """Whether x carries a forward-mode derivative (looked up only inside a dual level, where the module tells)."""
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(x).tangent is not None


def check_written(name, t):
    """Refuse a (n, heads, dim) tensor with contiguous rows as an output if autograd follows it or its rows overlap."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} cannot be a tensor that requires a gradient")
    n, heads, dim = t.shape
    if (n > 1 and abs(t.stride(0)) < dim) or (heads > 1 and abs(t.stride(1)) < dim):
        raise ValueError(f"the rows of {name} overlap: shape {tuple(t.shape)}, strides {t.stride()}")


def _inverse_frequencies(dim, base, scaling):
    """([dim/2] angles per position in float64, factor of the rotated vector)."""
    i = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    if scaling is None:
        return base ** -i, 1.0
    scaling = dict(scaling)
    kind = scaling.pop("type", None)
    known = {"linear": ("factor",), "ntk": ("factor",),
             "yarn": ("factor", "original_max_position", "beta_fast", "beta_slow", "attention_factor"),
             "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position")}
    if kind not in known:
        raise ValueError(f"scaling type must be one of {sorted(known)}, got {kind!r}")
    extra = set(scaling) - set(known[kind])
    if extra:
        raise ValueError(f"unknown entries for {kind} scaling: {sorted(extra)}")
    if not float(scaling.get("factor", 0.0)) > 0.0:
        raise ValueError("scaling needs a positive factor")
    factor = float(scaling["factor"])
    if kind == "linear":
        return base ** -i / factor, 1.0
    if kind == "ntk":
        if dim == 2:
            raise ValueError("ntk scaling needs a rotary dimension above 2")
        return (base * factor ** (dim / (dim - 2))) ** -i, 1.0
    w = base ** -i
    if not scaling.get("original_max_position", 0) > 0:
        raise ValueError(f"{kind} scaling needs original_max_position")
    old = float(scaling["original_max_position"])
    if kind == "llama3":
        low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
        if not high > low > 0.0:
            raise ValueError("llama3 scaling needs high_freq_factor > low_freq_factor > 0")
        wave = 2 * math.pi / w
        smooth = (old / wave - low) / (high - low)
        mid = (1 - smooth) * w / factor + smooth * w
        return torch.where(wave > old / low, w / factor, torch.where(wave < old / high, w, mid)), 1.0
    fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
    if not (fast > 0.0 and slow > 0.0 and base > 1.0):
        raise ValueError("yarn scaling needs positive betas and a base above 1")
    at = lambda turns: dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    first, last = max(0, math.floor(at(fast))), min(dim - 1, math.ceil(at(slow)))
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0, 1)
    attention = scaling.get("attention_factor")
    if attention is None:
        attention = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return w / factor * ramp + w * (1 - ramp), float(attention)


class Rotary:
    """Rotation of the first `dim` coordinates of a head by its position.

    Pair i is (x[i], x[i + dim/2]), or (x[2i], x[2i+1]) if `interleaved`, and turns by
    position * base^(-2i/dim).  `scaling` for contexts longer than a model was trained on:
    None, or a dict with "type" and

      linear   factor                       all angles divided by it
      ntk      factor                       base * factor^(dim/(dim-2))
      yarn     factor, original_max_position, [beta_fast 32, beta_slow 1, attention_factor]
               slow pairs divided, fast ones kept, a ramp between; the vector is multiplied
               by attention_factor (0.1 ln(factor) + 1)
      llama3   factor, original_max_position, [low_freq_factor 1, high_freq_factor 4]

    Angles are 64-bit fractions of a turn, so a position's phase is exact however far it is.
    """

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling=None, device=None):
        if dim < 2 or dim % 2 or dim > 8192:
            raise ValueError(f"the rotary dimension must be even, from 2 to 8192, got {dim}")
        if not base > 0.0:
            raise ValueError("base must be positive")
        self.dim, self.base, self.interleaved = int(dim), float(base), bool(interleaved)
        self.scaling = None if scaling is None else dict(scaling)
        self.inv_freq, self.factor = _inverse_frequencies(self.dim, self.base, self.scaling)
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise ValueError(f"Rotary needs a CUDA device, got {device}")
        self._L = _lib.load()
        turns = ((self.inv_freq.numpy() / (2 * math.pi)) % 1.0 * 2.0 ** 64).astype(np.uint64)
        self._turns = torch.from_numpy(turns.view(np.int64)).to(device)
        self.device = self._turns.device
        self._index = self.device.index
        self._desc = _lib.RotaryDesc(self._turns.data_ptr(), self.factor, self.dim, int(self.interleaved))
        self._ref = C.addressof(self._desc)

    def __reduce__(self):  # copies and pickles make a new one: the descriptor holds device addresses
        return Rotary, (self.dim, self.base, self.interleaved, self.scaling, str(self.device))

    def __call__(self, x: torch.Tensor, positions: torch.Tensor, out: torch.Tensor = None) -> torch.Tensor:
        """x [tokens, heads, dim >= self.dim] (float32, float16 or bfloat16; any strides, the last one 1), positions
        [tokens] (int32 or int64) -> the same shape and type.  `out` may be x (in place).  Differentiable in x (without
        `out`), backwards and forwards.  A given `out` is marked as modified, as PyTorch's own in-place operations do."""
        if (x.requires_grad and torch.is_grad_enabled()) or _has_tangent(x):
            if out is not None:
                raise ValueError("out cannot be given for an x that requires a gradient or has a tangent")
            return _Rotate.apply(x, positions, self)
        return self._apply(x.detach(), positions, out, 0)

    def _apply(self, x, positions, out, inverse):
        kind = TYPES.get(x.dtype)
        if x.dim() != 3 or kind is None or x.get_device() != self._index:
            raise ValueError(f"x must be (tokens, heads, dim) float32, float16 or bfloat16 on {self.device}, got {tuple(x.shape)} "
                             f"{x.dtype} on {x.device}")
        n, heads, dim = x.shape
        if dim < self.dim:
            raise ValueError(f"x has {dim} coordinates a head, the rotation {self.dim}")
        wide = positions.dtype is torch.int64
        if positions.dim() != 1 or len(positions) != n or not (wide or positions.dtype is torch.int32) or positions.get_device() != self._index:
            raise ValueError(f"positions must be ({n},) int32 or int64 on {self.device}, got {tuple(positions.shape)} "
                             f"{positions.dtype} on {positions.device}")
        xs = x.stride()
        if xs[2] != 1 and dim > 1:
            x = x.contiguous()
            xs = x.stride()
        given = out is not None
        if not given:
            out = torch.empty((n, heads, dim), dtype=x.dtype, device=self.device)
        elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or (dim > 1 and out.stride(2) != 1):
            raise ValueError("out must have the shape, type and device of x and contiguous rows")
        else:
            check_written("out", out)
        if not positions.is_contiguous():
            positions = positions.contiguous()
        ys = out.stride()
        if self._L.adaptq_rotary_apply(self._ref, x.data_ptr(), xs[0], xs[1], out.data_ptr(), ys[0], ys[1], kind, positions.data_ptr(), wide,
                                       n, heads, dim, inverse, self._index, current_stream(self._index)):
            raise RuntimeError(_lib.last_error())
        if given:
            increment_version(out)
        return out


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, rotary, inverse=0):
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        return rotary._apply(x, positions, None, inverse)

    @staticmethod
    def backward(ctx, grad):
        positions, = ctx.saved_tensors
        if (grad.requires_grad and torch.is_grad_enabled()) or _has_tangent(grad):  # a derivative of the gradient is wanted
            return _Rotate.apply(grad, positions, ctx.rotary, 1 - ctx.inverse), None, None, None
        return ctx.rotary._apply(grad, positions, None, 1 - ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):  # the rotation is linear: the tangent turns as x does
        positions, = ctx.saved_tensors
        return _Rotate.apply(tangent, positions, ctx.rotary, ctx.inverse)
