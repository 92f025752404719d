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
from torch.autograd import forward_ad
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
    dim: int = dataclasses.field(init=False)        # elements of a head that are rotated

    def __post_init__(self):
        w, h, a = self.inv_freq, self.half_turns, self.axis
        if w.dim() != 1 or h.shape != w.shape or h.dtype is not torch.float64 or h.device != w.device or not h.is_contiguous() \
                or (a is not None and (a.shape != w.shape or a.dtype is not torch.int32 or a.device != w.device or not a.is_contiguous())):
            raise ValueError("rotary: expected frequencies as rotary_frequencies makes them")
        object.__setattr__(self, "dim", 2 * w.shape[0])

    def to(self, device) -> "Rotary":
        move = lambda t: None if t is None else t.to(device)
        return dataclasses.replace(self, inv_freq=move(self.inv_freq), half_turns=move(self.half_turns), axis=move(self.axis))


_LARGEST = 1e30          # of an amplitude, which the kernels hold in 32 bits
# What a dictionary may hold: the kind, what belongs to the caller's other arguments or says nothing about angles, and the keys of any kind (a kind passes
# over those of the others, as configurations carry them along).  A key that is not here might change angles in a way that is not followed.
_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "max_position_embeddings", "finetuned", "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor",
         "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"}


def _positive(scaling: dict, name: str) -> Optional[float]:
    """The number under ``name``, or None where there is none."""
    if scaling.get(name) is None:
        return None
    value = float(scaling[name])
    if not (math.isfinite(value) and value > 0):
        raise ValueError(f"rotary scaling: {name} must be positive, got {scaling[name]}")
    return value


def _need(scaling: dict, name: str, kind: str) -> float:
    value = _positive(scaling, name)
    if value is None:
        raise ValueError(f"rotary scaling {kind!r} needs {name!r}")
    return value


def _check_scaling(scaling: dict, theta: float) -> str:
    """The kind of scaling; raises ``ValueError`` for what would be passed over."""
    unknown = [k for k, v in scaling.items() if k not in _KEYS and v is not None]
    if unknown:
        raise ValueError(f"rotary scaling: unknown keys {unknown}")
    kind = scaling.get("rope_type") or scaling.get("type")
    if kind is None:
        if scaling.get("factor") is not None:
            raise ValueError("rotary scaling: a factor needs a 'rope_type'")
        kind = "default"
    if scaling.get("rope_theta") is not None and float(scaling["rope_theta"]) != theta:
        raise ValueError(f"rotary scaling: rope_theta {scaling['rope_theta']} is not theta {theta}")
    return kind


def _yarn_amplitude(scaling: dict, factor: float) -> float:
    amplitude = scaling.get("attention_factor")
    if amplitude is None:
        over, under = (_positive(scaling, name) if scaling.get(name) else None for name in ("mscale", "mscale_all_dim"))     # 0: not given
        log = math.log(factor) if factor > 1 else 0.0
        amplitude = 0.1 * log + 1.0 if over is None or under is None else (0.1 * over * log + 1.0) / (0.1 * under * log + 1.0)
    amplitude = float(amplitude)
    if not abs(amplitude) <= _LARGEST:
        raise ValueError(f"rotary scaling: amplitude {amplitude} is not finite, or beyond {_LARGEST}")
    return amplitude


def _axis_frequencies(dim: int, theta: float, scaling: dict) -> Tuple[torch.Tensor, float]:
    kind = _check_scaling(scaling, theta)
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
    fast, slow = (_positive(scaling, name) if scaling.get(name) else turns for name, turns in (("beta_fast", 32.0), ("beta_slow", 1.0)))     # 0: not given

    def pair_with(turns: float) -> float:
        return dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))

    low, high = pair_with(fast), pair_with(slow)
    if scaling.get("truncate", True):           # the ramp from whole pair to whole pair
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return (1.0 - ramp) * inv + ramp * inv / factor, _yarn_amplitude(scaling, factor)


def rotary_frequencies(dim: int, theta: float = 10000.0, *, axes: Optional[Sequence[int]] = None, scaling: Optional[dict] = None,
                       interleaved: bool = False, device=None) -> Rotary:
    """Frequencies ``theta^(-2 j / dim)`` of ``dim / 2`` pairs.

    ``axes``: the rotated elements of each position axis (``(16, 56, 56)`` for a video's frames, rows and columns; they sum to
    ``dim`` and every axis starts with its fastest pair).  ``scaling``: a model configuration's dictionary, ``rope_type`` one of
    ``linear`` and ``ntk`` (``factor``), ``llama3`` (``factor``, ``low_freq_factor``, ``high_freq_factor``,
    ``original_max_position_embeddings``), ``yarn`` (``factor``, ``original_max_position_embeddings``; optionally ``beta_fast``, ``beta_slow``,
    ``truncate``, ``mscale`` with ``mscale_all_dim``, ``attention_factor``); it applies to every axis.  Keys that no kind knows, a factor without a kind
    and a ``rope_theta`` other than ``theta`` are refused."""
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


def check_arguments(q, k, positions, rotary: Rotary) -> Tuple[int, int, int]:
    """Raises ``ValueError`` where the operands do not belong together; returns the positions' strides over samples, axes and tokens.
    (A call for a few tokens takes the host longer than the device, so what is right is found to be so with few look-ups.)"""
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary: expected the frequencies that rotary_frequencies returns")
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"expected [batch, heads, tokens, head_dim], got q {tuple(q.shape)}" + ("" if k is None else f", k {tuple(k.shape)}"))
    B, _, S, D = q.shape
    device = q.get_device()
    if k is not None:
        Bk, _, Sk, Dk = k.shape
        if Bk != B or Sk != S or Dk != D or k.dtype is not q.dtype or k.get_device() != device:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} on {q.device} and k {tuple(k.shape)} {k.dtype} on {k.device} do not belong together")
    if not q.dtype.is_floating_point:
        raise ValueError(f"q: expected a floating type, got {q.dtype}")
    if rotary.dim > D:
        raise ValueError(f"{rotary.dim} elements to rotate in heads of {D}")
    if rotary.inv_freq.get_device() != device:
        raise ValueError(f"rotary frequencies on {rotary.inv_freq.device}, queries on {q.device}")
    if (positions.dtype is not torch.int32 and positions.dtype is not torch.int64) or positions.get_device() != device:
        raise ValueError(f"positions: expected int32 or int64 on {q.device}, got {positions.dtype} on {positions.device}")
    A, shape, stride = rotary.num_axes, tuple(positions.shape), positions.stride()
    if A == 1:
        if shape == (S,):
            return 0, 0, stride[0]
        if shape == (B, S) or shape == (1, S):
            return (stride[0] if shape[0] > 1 else 0), 0, stride[1]
    if shape == (A, S):
        return 0, stride[0], stride[1]
    if shape == (B, A, S) or shape == (1, A, S):
        return (stride[0] if shape[0] > 1 else 0), stride[1], stride[2]
    want = "[tokens] or [batch, tokens]" if A == 1 else f"[{A}, tokens] or [batch, {A}, tokens]"
    raise ValueError(f"positions: expected {want} for {S} tokens of {B} samples, got {shape}")


def by_axis(positions, num_axes: int):
    """Positions that :func:`check_arguments` has taken as ``[1 or batch, axes, tokens]``, for the plain path."""
    if positions.dim() == 3:
        return positions
    if num_axes > 1:
        return positions[None]
    return positions[None, None] if positions.dim() == 1 else positions[:, None]


def check_norm(q, k, q_weight, k_weight, eps) -> None:
    if k is None:
        raise ValueError("qk_norm_rotary: expected queries and keys")
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps: expected a number of 0 or more, got {eps}")
    for x, w, n in ((q, q_weight, "q_weight"), (k, k_weight, "k_weight")):
        if w.dim() != 1 or w.shape[0] != x.shape[3] or w.dtype is not x.dtype or w.get_device() != x.get_device():
            raise ValueError(f"{n}: expected [{x.shape[3]}] {x.dtype} on {x.device}, got {tuple(w.shape)} {w.dtype} on {w.device}")


def supported(q) -> bool:
    return q.dtype in _DTYPES and q.shape[3] % 2 == 0 and q.shape[3] <= MAX_HEAD_DIM


# ------------------------------------------------------------------------------------------------ native calls

_HEAD = struct.Struct("@lll iiii iiii PP 6l PP 6l P 3l PP ff PP")        # everything that the forward kernels read
_ARGS = struct.Struct("@lll iiii iiii PP 6l PP 6l P 3l PP ff PP PP 6l PP P l")
_NO_BACKWARD = bytes(_ARGS.size - _HEAD.size)


def _rows(t):
    """Operand with a contiguous last dimension (its other strides are free)."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _pack(q, k, out_q, out_k, positions, pos_stride, rotary, transpose, eps, q_weight, k_weight):
    """The arguments that the forward kernels read; ``q`` or ``k`` may be None."""
    some = k if q is None else q
    B, _, S, D = some.shape
    hq = hk = 0
    pq = pk = oq = ok = 0
    sq = sk = tq = tk = (0, 0, 0, 0)
    if q is not None:
        hq, pq, oq, sq, tq = q.shape[1], q.data_ptr(), out_q.data_ptr(), q.stride(), out_q.stride()
    if k is not None:
        hk, pk, ok, sk, tk = k.shape[1], k.data_ptr(), out_k.data_ptr(), k.stride(), out_k.stride()
    return _HEAD.pack(_ARGS.size, B, S, hq, hk, D, rotary.dim >> 1, _DTYPES[some.dtype], rotary.interleaved, transpose, positions.dtype is torch.int64,
                      pq, pk, sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], oq, ok, tq[0], tq[1], tq[2], tk[0], tk[1], tk[2], positions.data_ptr(),
                      *pos_stride, rotary.half_turns.data_ptr(), 0 if rotary.axis is None else rotary.axis.data_ptr(), rotary.amplitude, eps,
                      0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr())


def _ordered(x, token_major: bool):
    """An empty tensor of ``x``'s shape in the given order of heads and tokens: the gradient of a token-major projection's view then needs
    no transposition."""
    B, H, S, D = x.shape
    return x.new_empty_strided((B, H, S, D), (S * H * D, D, H * D, 1)) if token_major else x.new_empty((B, H, S, D))


def _token_major(x) -> bool:
    return x.stride(1) < x.stride(2)


def _forward(q, k, positions, pos_stride, freqs):
    q = _rows(q)
    out_q, out_k = q.new_empty(q.shape), None
    if k is not None:
        k = _rows(k)
        out_k = k.new_empty(k.shape)
    some_q, some_k = q.numel() > 0, k is not None and k.numel() > 0
    if some_q or some_k:
        call("tt_rotary", _pack(q if some_q else None, k if some_k else None, out_q, out_k, positions, pos_stride, freqs, False, 0.0, None, None)
             + _NO_BACKWARD, stream())
    return out_q, out_k


def _rotary_backward(ctx, gq, gk=None):
    positions, = ctx.saved_tensors
    grads = []
    for g, need, order in zip((gq, gk), ctx.needs_input_grad, ctx.token_major):
        grads.append((_rows(g), _ordered(g, order)) if need and g is not None else (None, None))
    (gq, dq), (gk, dk) = grads
    some_q, some_k = gq is not None and gq.numel() > 0, gk is not None and gk.numel() > 0
    if some_q or some_k:
        with on_device(positions):
            call("tt_rotary", _pack(gq if some_q else None, gk if some_k else None, dq, dk, positions, ctx.pos_stride, ctx.freqs, True, 0.0, None, None)
                 + _NO_BACKWARD, stream())
    return dq, dk, None, None, None


_rotary_backward_once = once_differentiable(_rotary_backward)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, pos_stride, freqs):
        ctx.freqs, ctx.pos_stride = freqs, pos_stride
        ctx.save_for_backward(positions)
        ctx.token_major = (_token_major(q), k is not None and _token_major(k))
        out = _forward(q, k, positions, pos_stride, freqs)
        return out[0] if k is None else out

    @staticmethod
    def backward(ctx, *grads):
        # the wrapper, which a second derivative would need to fail in, costs the host 5 us of a first one
        return (_rotary_backward_once if torch.is_grad_enabled() else _rotary_backward)(ctx, *grads)


def rotary(q, k, positions, pos_stride, freqs):
    with on_device(q):
        # (under a forward-mode level operands may have tangents, which the autograd function refuses and a kernel alone would lose)
        if forward_ad._current_level >= 0 or (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))):
            out = _Rotary.apply(q, k, positions, pos_stride, freqs)
            return (out, None) if k is None else out
        return _forward(q, k, positions, pos_stride, freqs)


def _norm_forward(q, k, q_weight, k_weight, positions, pos_stride, freqs, eps):
    out_q, out_k = q.new_empty(q.shape), k.new_empty(k.shape)
    some_q, some_k = q.numel() > 0, k.numel() > 0
    if some_q or some_k:
        call("tt_norm_rotary_fwd", _pack(q if some_q else None, k if some_k else None, out_q, out_k, positions, pos_stride, freqs, False, eps, q_weight,
                                         k_weight) + _NO_BACKWARD, stream())
    return out_q, out_k


_TAIL = struct.Struct("@PP 6l PP P l")


def _norm_backward(ctx, gq, gk):
    q, k, q_weight, k_weight, positions = ctx.saved_tensors
    with on_device(q):
        gq, gk = _rows(gq), _rows(gk)
        dq, dk = _ordered(q, _token_major(q)), _ordered(k, _token_major(k))
        dqw, dkw = q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)
        some_q, some_k = q.numel() > 0, k.numel() > 0
        for some, dw in ((some_q, dqw), (some_k, dkw)):
            if not some:
                dw.zero_()
        if some_q or some_k:
            head = _pack(q if some_q else None, k if some_k else None, dq, dk, positions, ctx.pos_stride, ctx.freqs, False, ctx.eps, q_weight, k_weight)
            grads = (gq.data_ptr(), gk.data_ptr(), *gq.stride()[:3], *gk.stride()[:3], dqw.data_ptr(), dkw.data_ptr())
            size = _lib.lib().tt_rotary_partial_floats(head + _TAIL.pack(*grads, 0, 0))         # by the gradients' alignment too
            partials = q.new_empty((max(size, 1),), dtype=torch.float32)
            call("tt_norm_rotary_bwd", head + _TAIL.pack(*grads, partials.data_ptr(), size), stream())
    a, b, c, d = ctx.needs_input_grad[:4]
    return dq if a else None, dk if b else None, dqw if c else None, dkw if d else None, None, None, None, None


_norm_backward_once = once_differentiable(_norm_backward)


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, pos_stride, freqs, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.pos_stride, ctx.freqs, ctx.eps = pos_stride, freqs, eps
        return _norm_forward(q, k, q_weight, k_weight, positions, pos_stride, freqs, eps)

    @staticmethod
    def backward(ctx, gq, gk):
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, gq, gk)


def qk_norm_rotary(q, k, q_weight, k_weight, positions, pos_stride, freqs, eps):
    with on_device(q):
        q, k, q_weight, k_weight = _rows(q), _rows(k), q_weight.contiguous(), k_weight.contiguous()
        if forward_ad._current_level >= 0 or \
                (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or q_weight.requires_grad or k_weight.requires_grad)):
            return _NormRotary.apply(q, k, q_weight, k_weight, positions, pos_stride, freqs, float(eps))
        return _norm_forward(q, k, q_weight, k_weight, positions, pos_stride, freqs, float(eps))
