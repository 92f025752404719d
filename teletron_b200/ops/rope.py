"""Rotary positions of queries and keys: interleaved and half layouts, part of the head, several position axes, frequencies
scaled for long contexts; alone or behind an RMS norm of every head (``csrc/rotary.cu``).

The reference rotates interleaved pairs by tables that it stores in fp32 (``teletron/models/hunyuanvideo/layers.py:209-252``,
``teletron/models/dit/dit_attention.py:265-273``); its text encoders bring the half layout and their own scaling with them
(``teletron/models/hunyuanvideo/text_encoder.py``).  Here the angles are formed in 64 bits from integer positions where they are used, so no table
is stored or read.
"""

from __future__ import annotations

import dataclasses
import math
import struct
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import call, on_device, stream

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_HEAD_DIM = 256


@dataclasses.dataclass(frozen=True)
class Rotary:
    """Frequencies of a rotation, as :func:`rotary_frequencies` makes them.

    ``inv_freq``: radians per position of every pair, 64 bits; ``half_turns``: the same in units of pi; ``axis``: position axis of
    every pair (int32) or None where there is one; ``amplitude``: factor on the rotated elements; ``interleaved``: pairs are
    neighbours ``(2 p, 2 p + 1)`` instead of halves ``(p, P + p)``."""
    inv_freq: torch.Tensor
    half_turns: torch.Tensor
    axis: Optional[torch.Tensor]
    num_axes: int
    amplitude: float
    interleaved: bool

    @property
    def dim(self) -> int:
        """Elements of a head that are rotated."""
        return 2 * self.inv_freq.shape[0]

    def to(self, device) -> "Rotary":
        move = lambda t: None if t is None else t.to(device)
        return dataclasses.replace(self, inv_freq=move(self.inv_freq), half_turns=move(self.half_turns), axis=move(self.axis))


def _need(scaling: dict, name: str, kind: str) -> float:
    if name not in scaling:
        raise ValueError(f"rotary scaling {kind!r} needs {name!r}")
    value = float(scaling[name])
    if not (math.isfinite(value) and value > 0):
        raise ValueError(f"rotary scaling: {name} must be positive, got {scaling[name]}")
    return value


def _axis_frequencies(dim: int, theta: float, scaling: dict) -> Tuple[torch.Tensor, float]:
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    j = torch.arange(0, dim, 2, dtype=torch.float64)
    inv = theta ** (-j / dim)
    if kind in ("default", "none"):
        return inv, 1.0
    if kind not in ("linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown rotary scaling {kind!r} (linear, ntk, llama3, yarn)")
    factor = _need(scaling, "factor", kind)
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "ntk":           # a larger base instead: the slowest pair is stretched by the factor, the fastest not at all
        if dim <= 2:
            raise ValueError("rotary scaling 'ntk' needs more than one pair per axis")
        return (theta * factor ** (dim / (dim - 2))) ** (-j / dim), 1.0
    context = _need(scaling, "original_max_position_embeddings", kind)
    if kind == "llama3":        # by the turns a pair makes over the original context: many are kept, few are stretched
        low, high = _need(scaling, "low_freq_factor", kind), _need(scaling, "high_freq_factor", kind)
        if high <= low:
            raise ValueError("rotary scaling 'llama3': high_freq_factor must exceed low_freq_factor")
        keep = ((context * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return keep * inv + (1.0 - keep) * inv / factor, 1.0
    if theta <= 1.0:
        raise ValueError("rotary scaling 'yarn' needs a theta above 1")
    fast, slow = float(scaling.get("beta_fast") or 32.0), float(scaling.get("beta_slow") or 1.0)

    def pair_with(turns: float) -> float:
        return dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = max(math.floor(pair_with(fast)), 0), min(math.ceil(pair_with(slow)), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    amplitude = scaling.get("attention_factor")
    if amplitude is None:
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return (1.0 - ramp) * inv + ramp * inv / factor, float(amplitude)


def rotary_frequencies(dim: int, theta: float = 10000.0, *, axes: Optional[Sequence[int]] = None, scaling: Optional[dict] = None,
                       interleaved: bool = False, device=None) -> Rotary:
    """Frequencies ``theta^(-2 j / dim)`` of ``dim / 2`` pairs.

    ``axes``: the rotated elements of each position axis (``(16, 56, 56)`` for a video's frames, rows and columns; they sum to
    ``dim`` and every axis starts with its fastest pair).  ``scaling``: a model configuration's dictionary, ``rope_type`` one of
    ``linear`` and ``ntk`` (``factor``), ``llama3`` (``factor``, ``low_freq_factor``, ``high_freq_factor``,
    ``original_max_position_embeddings``), ``yarn`` (``factor``, ``original_max_position_embeddings``; optionally ``beta_fast``, ``beta_slow``,
    ``attention_factor``); it applies to every axis."""
    dims = [int(dim)] if axes is None else [int(a) for a in axes]
    if not dims or any(d <= 0 or d % 2 for d in dims) or sum(dims) != dim:
        raise ValueError(f"rotary dims must be positive, even and sum to {dim}, got {dims}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"theta must be positive, got {theta}")
    parts = [_axis_frequencies(d, float(theta), scaling or {}) for d in dims]
    inv = torch.cat([p[0] for p in parts])
    axis = None
    if len(dims) > 1:
        axis = torch.cat([torch.full((d // 2,), a, dtype=torch.int32) for a, d in enumerate(dims)])
    rot = Rotary(inv, inv / math.pi, axis, len(dims), parts[0][1], bool(interleaved))
    return rot if device is None else rot.to(device)


def check_arguments(q, k, positions, rotary: Rotary) -> torch.Tensor:
    """Raises ``ValueError`` where the operands do not belong together; returns the positions as ``[1 or batch, axes, tokens]``."""
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary: expected the frequencies that rotary_frequencies returns")
    for t, n in ((q, "q"), (k, "k")):
        if t is None and n == "k":
            continue
        if t.dim() != 4:
            raise ValueError(f"{n}: expected [batch, heads, tokens, head_dim], got {tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != q.device or (t.shape[0], t.shape[2], t.shape[3]) != (q.shape[0], q.shape[2], q.shape[3]):
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} on {q.device} and k {tuple(t.shape)} {t.dtype} on {t.device} do not belong together")
    if not q.dtype.is_floating_point:
        raise ValueError(f"q: expected a floating type, got {q.dtype}")
    if rotary.dim > q.shape[3]:
        raise ValueError(f"{rotary.dim} elements to rotate in heads of {q.shape[3]}")
    if rotary.inv_freq.device != q.device:
        raise ValueError(f"rotary frequencies on {rotary.inv_freq.device}, queries on {q.device}")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != q.device:
        raise ValueError(f"positions: expected int32 or int64 on {q.device}, got {positions.dtype} on {positions.device}")
    B, S, A = q.shape[0], q.shape[2], rotary.num_axes
    p = positions
    if A == 1 and p.dim() in (1, 2):
        p = p.view(1, 1, -1) if p.dim() == 1 else p[:, None]
    elif A > 1 and p.dim() == 2:
        p = p[None]
    if p.dim() != 3 or p.shape[0] not in (1, B) or p.shape[1:] != (A, S):
        want = "[tokens] or [batch, tokens]" if A == 1 else f"[{A}, tokens] or [batch, {A}, tokens]"
        raise ValueError(f"positions: expected {want} for {S} tokens of {B} samples, got {tuple(positions.shape)}")
    return p


def check_weights(q, k, q_weight, k_weight) -> None:
    for x, w, n in ((q, q_weight, "q_weight"), (k, k_weight, "k_weight")):
        if w.shape != (x.shape[3],) or w.dtype != x.dtype or w.device != x.device:
            raise ValueError(f"{n}: expected [{x.shape[3]}] {x.dtype} on {x.device}, got {tuple(w.shape)} {w.dtype} on {w.device}")


def supported(q) -> bool:
    return q.dtype in _DTYPES and q.shape[3] % 2 == 0 and q.shape[3] <= MAX_HEAD_DIM


# ------------------------------------------------------------------------------------------------ native calls

_ARGS = struct.Struct("@lll iiii iiii PP 6l PP 6l P 3l PP ff PP PP 6l PP P l")
_NONE3 = (0, 0, 0)


def _rows(t):
    """Operand with a contiguous last dimension (its other strides are free)."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _strides(t):
    return _NONE3 if t is None else t.stride()[:3]


def _address(t):
    return 0 if t is None else t.data_ptr()


def _native(fn, q, k, out_q, out_k, positions, rotary, *, transpose=False, eps=0.0, weights=(None, None), grads=(None, None), dweights=(None, None),
            partials=None):
    B, _, S, D = q.shape if q is not None else k.shape
    dtype = (q if q is not None else k).dtype
    packed = _ARGS.pack(
        _ARGS.size, B, S, 0 if q is None else q.shape[1], 0 if k is None else k.shape[1], D, rotary.dim // 2,
        _DTYPES[dtype], rotary.interleaved, transpose, positions.dtype == torch.int64,
        _address(q), _address(k), *_strides(q), *_strides(k), _address(out_q), _address(out_k), *_strides(out_q), *_strides(out_k),
        positions.data_ptr(), 0 if positions.shape[0] == 1 else positions.stride(0), positions.stride(1), positions.stride(2),
        rotary.half_turns.data_ptr(), _address(rotary.axis), rotary.amplitude, eps, _address(weights[0]), _address(weights[1]),
        _address(grads[0]), _address(grads[1]), *_strides(grads[0]), *_strides(grads[1]), _address(dweights[0]), _address(dweights[1]),
        _address(partials), 0 if partials is None else partials.numel())
    if fn is None:
        return packed
    call(fn, packed, stream())


def _head_major(t):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _like(x):
    """An output in ``x``'s order of heads and tokens, so that the gradient of a token-major projection needs no transposition."""
    B, H, S, D = x.shape
    if x.stride(1) < x.stride(2):
        return torch.empty(B, S, H, D, dtype=x.dtype, device=x.device).transpose(1, 2)
    return torch.empty(B, H, S, D, dtype=x.dtype, device=x.device)


def _rotate(q, k, positions, rotary, transpose, make):
    """``k`` None: queries only."""
    ins = [None if t is None else _rows(t) for t in (q, k)]
    outs = [None if t is None else make(t) for t in (q, k)]
    if any(t is not None and t.numel() for t in ins):
        _native("tt_rotary", *[t if t is not None and t.numel() else None for t in ins], *outs, positions, rotary, transpose=transpose)
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, rotary):
        ctx.rotary = rotary
        ctx.save_for_backward(positions)
        ctx.token_major = [t is not None and t.stride(1) < t.stride(2) for t in (q, k)]
        out = _rotate(q, k, positions, rotary, False, _head_major)
        return out[0] if k is None else tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk=None):
        positions, = ctx.saved_tensors
        grads = [g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad)]
        order = iter([t for t, g in zip(ctx.token_major, grads) if g is not None])

        def make(g):
            B, H, S, D = g.shape
            if next(order):
                return torch.empty(B, S, H, D, dtype=g.dtype, device=g.device).transpose(1, 2)
            return _head_major(g)

        if all(g is None for g in grads):
            return None, None, None, None
        with on_device(positions):
            dq, dk = _rotate(*grads, positions, ctx.rotary, True, make)
        return dq, dk, None, None


def rotary(q, k, positions, freqs):
    with on_device(q):
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            out = _Rotary.apply(q, k, positions, freqs)
            return (out, None) if k is None else out
        return tuple(_rotate(q, k, positions, freqs, False, _head_major))


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, freqs, eps):
        q, k, q_weight, k_weight = _rows(q), _rows(k), q_weight.contiguous(), k_weight.contiguous()
        out = [_head_major(q), _head_major(k)]
        if out[0].numel() or out[1].numel():
            _native("tt_norm_rotary_fwd", *[t if t.numel() else None for t in (q, k)], *out, positions, freqs, eps=eps, weights=(q_weight, k_weight))
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.freqs, ctx.eps = freqs, eps
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        with on_device(q):
            gq, gk = _rows(gq), _rows(gk)
            dq, dk = _like(q), _like(k)
            dqw, dkw = torch.empty_like(q_weight), torch.empty_like(k_weight)
            ins, outs, grads, weights, dws = [], [], [], [], []
            for x, dx, g, w, dw in ((q, dq, gq, q_weight, dqw), (k, dk, gk, k_weight, dkw)):
                some = x.numel() > 0
                if not some:
                    dw.zero_()
                for into, t in zip((ins, outs, grads, weights, dws), (x, dx, g, w, dw)):
                    into.append(t if some else None)
            if ins[0] is not None or ins[1] is not None:
                kw = dict(eps=ctx.eps, weights=weights, grads=grads, dweights=dws)
                n = _lib.lib().tt_rotary_partial_floats(_native(None, *ins, *outs, positions, ctx.freqs, **kw))
                partials = torch.empty(max(n, 1), dtype=torch.float32, device=q.device)
                _native("tt_norm_rotary_bwd", *ins, *outs, positions, ctx.freqs, partials=partials, **kw)
        need = ctx.needs_input_grad
        return tuple(t if n else None for t, n in zip((dq, dk, dqw, dkw), need)) + (None, None, None)


def qk_norm_rotary(q, k, q_weight, k_weight, positions, freqs, eps):
    with on_device(q):
        return _NormRotary.apply(q, k, q_weight, k_weight, positions, freqs, float(eps))
