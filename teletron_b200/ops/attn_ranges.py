"""Attention in which every query sees one run of the keys (``csrc/attn_ranges_*.cu``).

Causal, prefix and document masks, padded batches and caches in use up to a length all let a query see one run of keys.  A
:class:`KeyRanges` holds the runs and what the kernels need to skip and to mask by tiles; it is made once for a batch and shared by its
layers.  The reference passes no mask to its attention at all (``teletron/models/dit/dit_attention.py:311-313``) and leaves
the text encoders' masks and biases to their package (``teletron/models/hunyuanvideo/text_encoder.py``).
"""

from __future__ import annotations

import ctypes
import dataclasses
import math
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import c_int, c_long, call, on_device, ptr, stream
from .gemm_tcgen05 import status_tensor

TILE = 128
MAX_DISTANCE = 1024
MAX_BATCH = MAX_HEADS = 65535
_LARGEST = 1e30
MAX_LEN = 1 << 30           # of queries and of keys
_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


@dataclasses.dataclass(frozen=True, eq=False)
class KeyRanges:
    """Runs of keys ``[first, behind)`` that the queries of a batch see (int32 ``[batch, q_len]`` both; 0, 0: none).

    Made by :func:`key_ranges`; its tensors are not to be written to."""
    batch: int
    q_len: int
    kv_len: int
    first: torch.Tensor
    behind: torch.Tensor
    query_start: Optional[torch.Tensor]
    plan: Optional[torch.Tensor]
    causal: bool = False            # runs grow with the query: what the kernels begin with

    @property
    def device(self):
        return self.first.device


def _lengths(value, name: str, batch: int, device, per_document: Optional[int] = None):
    """An int, or per-sample integers, as ``(int or None, int32 tensor or None)``."""
    if value is None or isinstance(value, int):
        return value, None
    t = value if isinstance(value, torch.Tensor) else torch.tensor(value)
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name}: expected integers, got {t.dtype}")
    shapes = [(batch,)] + ([(batch, per_document)] if per_document is not None else [])
    if tuple(t.shape) not in shapes:
        raise ValueError(f"{name}: expected an int or one of the shapes {shapes}, got {tuple(t.shape)}")
    return None, _int32(t.to(device))


def _int32(t):
    """Lengths, offsets and positions in 32 bits; what lies beyond them is beyond every length too."""
    return (t if t.dtype is torch.int32 else t.clamp(-MAX_LEN, MAX_LEN).to(torch.int32)).contiguous()


def _runs(q_len, kv_len, batch, causal, documents, prefix_len, prefix, kv_valid_len, query_start, device):
    """The runs in torch operations: the definition, and the path without the native library's device."""
    i = torch.arange(q_len, device=device).expand(batch, q_len)
    at = i if query_start is None else i + query_start.long()[:, None]
    lo, hi, start, doc = torch.zeros_like(i), torch.full_like(i, kv_len), torch.zeros_like(i), None
    if kv_valid_len is not None:
        hi = torch.minimum(hi, kv_valid_len.long()[:, None].expand_as(hi))
    if documents is not None:
        off = documents.long().expand(batch, -1).contiguous()
        n = off.shape[1] - 1
        place = torch.searchsorted(off, i.contiguous(), right=True)
        inside = (place > 0) & (place <= n)
        doc = (place - 1).clamp(0, n - 1)
        start = off.gather(1, doc).clamp_min(0)
        lo = start
        hi = torch.where(inside, torch.minimum(hi, off.gather(1, doc + 1)), torch.zeros_like(hi))
    if causal:
        p = prefix_len or 0
        if prefix is not None:
            p = prefix.long()[:, None] if prefix.dim() == 1 else prefix.long().gather(1, doc)
            p = p.clamp_min(0)
        hi = torch.minimum(hi, torch.maximum(at + 1, start + p))
    none = lo >= hi
    return lo.masked_fill(none, 0).to(torch.int32), hi.masked_fill(none, 0).to(torch.int32)


def key_ranges(q_len: int, kv_len: Optional[int] = None, *, batch: int = 1, causal: bool = False, documents=None, prefix_len=None,
               kv_valid_len=None, query_start=None, device=None) -> KeyRanges:
    """The runs of keys that ``q_len`` queries of ``batch`` samples see among ``kv_len`` keys (default: as many as queries).

    * ``causal``: a query sees keys up to its own position, ``query_start`` (int or ``[batch]``, default 0) plus its index.
    * ``documents``: offsets of documents that are packed one after another, integers ``[n + 1]`` or ``[batch, n + 1]`` that do not
      decrease; a query sees its own document only, and nothing behind the last or ahead of the first.  A batch padded to the right is one
      document per sample, ``[[0, length], ...]``.  Needs ``q_len == kv_len`` and no ``query_start``.
    * ``prefix_len`` (int, ``[batch]`` or, with documents, ``[batch, n]``): that many first keys of the sample, or of each document, are
      seen by all of its queries.  Needs ``causal``.
    * ``kv_valid_len`` (int or ``[batch]``): keys from there on are seen by nobody (a cache that is not full).

    With ``causal`` and another number of keys than queries the positions have to be said, by ``query_start``."""
    q_len, kv_len, batch = int(q_len), int(q_len if kv_len is None else kv_len), int(batch)
    if q_len < 0 or kv_len < 0 or batch < 0:
        raise ValueError(f"key_ranges: negative sizes ({q_len} queries, {kv_len} keys, {batch} samples)")
    if max(q_len, kv_len) > MAX_LEN:
        raise ValueError(f"key_ranges: {q_len} queries and {kv_len} keys, at most {MAX_LEN} of each")
    for v in (documents, prefix_len, kv_valid_len, query_start):
        if device is None and isinstance(v, torch.Tensor):
            device = v.device
    device = torch.device("cpu" if device is None else device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if prefix_len is not None and not causal:
        raise ValueError("key_ranges: a prefix needs causal=True")
    if causal and q_len != kv_len and query_start is None:
        raise ValueError(f"key_ranges: {q_len} queries and {kv_len} keys: causal runs need query_start")
    n = None
    if documents is not None:
        if q_len != kv_len or query_start is not None:
            raise ValueError("key_ranges: documents need as many queries as keys and no query_start")
        documents = documents if isinstance(documents, torch.Tensor) else torch.tensor(documents)
        if documents.dtype not in (torch.int32, torch.int64) or documents.dim() not in (1, 2) or documents.shape[-1] < 2 \
                or (documents.dim() == 2 and documents.shape[0] != batch):
            raise ValueError(f"documents: expected integer offsets [n + 1] or [{batch}, n + 1], got {documents.dtype} {tuple(documents.shape)}")
        documents = _int32(documents.to(device))
        documents = documents[None] if documents.dim() == 1 else documents
        n = documents.shape[1] - 1
    prefix_len, prefix = _lengths(prefix_len, "prefix_len", batch, device, n)
    kv_valid_int, kv_valid = _lengths(kv_valid_len, "kv_valid_len", batch, device)
    start_int, start = _lengths(query_start, "query_start", batch, device)
    if prefix_len is not None:
        if prefix_len < 0:
            raise ValueError(f"prefix_len: {prefix_len} is negative")
        prefix_len = min(prefix_len, kv_len)
    if kv_valid_int is not None:
        kv_valid = torch.full((batch,), min(max(kv_valid_int, 0), kv_len), dtype=torch.int32, device=device)
    if start_int:
        start = torch.full((batch,), max(-MAX_LEN, min(MAX_LEN, start_int)), dtype=torch.int32, device=device)
    if device.type != "cuda" or not _lib.available() or min(q_len, kv_len, batch) == 0 or batch > MAX_BATCH:
        first, behind = _runs(q_len, kv_len, batch, causal, documents, prefix_len, prefix, kv_valid, start, device)
        return KeyRanges(batch, q_len, kv_len, first, behind, start, None, bool(causal))
    at = _layout(batch, q_len, kv_len)
    with torch.cuda.device(device):
        status_tensor(device)           # here, since in a captured attention it would be cleared by replays only
        plan = torch.empty(at.ints, dtype=torch.int32, device=device)
        call("tt_key_ranges", ptr(plan), c_int(batch), c_int(q_len), c_int(kv_len), c_int(causal), ptr(documents), c_int(n or 0),
             c_long(0 if documents is None or documents.shape[0] == 1 else documents.shape[1]), ptr(prefix),
             c_long(0 if prefix is None else prefix.stride(0)), c_int(prefix is not None and prefix.dim() == 2), c_int(prefix_len or 0),
             ptr(kv_valid), ptr(start), stream())
    rows = batch * q_len
    return KeyRanges(batch, q_len, kv_len, plan[at.first:at.first + rows].view(batch, q_len), plan[at.behind:at.behind + rows].view(batch, q_len),
                     start, plan, bool(causal))


class _Layout(ctypes.Structure):
    _fields_ = [(n, ctypes.c_long) for n in ("q_tiles", "dead", "k_tiles", "dirty", "first", "behind", "start", "ints")]


def _layout(batch, q_len, kv_len):
    at = _Layout()
    _lib.lib().tt_key_ranges_layout(c_int(batch), c_int(q_len), c_int(kv_len), ctypes.byref(at))
    return at


def check_arguments(q, k, v, ranges, scale, softcap, distance_bias) -> None:
    """Raises ``ValueError`` where the operands do not belong together."""
    if not isinstance(ranges, KeyRanges):
        raise ValueError("masked_attention: expected the runs that key_ranges returns")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"expected [batch, heads, tokens, head_dim], got q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    B, hq, n, D = q.shape
    Bk, hk, m, Dk = k.shape
    dtype, device = q.dtype, q.get_device()
    if k.shape != v.shape or Bk != B or Dk != D or hk == 0 or hq % hk:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if not dtype.is_floating_point or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != device or v.get_device() != device:
        raise ValueError(f"q {q.dtype} on {q.device}, k {k.dtype} on {k.device}, v {v.dtype} on {v.device} do not belong together")
    if ranges.batch != B or ranges.q_len != n or ranges.kv_len != m:
        raise ValueError(f"runs of {ranges.batch} x {ranges.q_len} queries and {ranges.kv_len} keys for {B} x {n} queries and {m} keys")
    if ranges.first.get_device() != device:
        raise ValueError(f"runs on {ranges.device}, queries on {q.device}")
    if scale is not None and not abs(scale) <= _LARGEST:
        raise ValueError(f"scale: {scale} is not finite, or beyond {_LARGEST}")
    # the kernels hold the cap, its inverse and scale / cap in 32 bits
    if softcap is not None and not (1 / _LARGEST <= softcap <= _LARGEST and (1.0 if scale is None else abs(scale)) <= _LARGEST * softcap):
        raise ValueError(f"softcap: expected a positive number or None, neither it nor the scale ({scale}) over it beyond {_LARGEST}, got {softcap}")
    if distance_bias is not None:
        if distance_bias.dim() != 2 or distance_bias.shape[0] != hq or distance_bias.shape[1] % 2 == 0:
            raise ValueError(f"distance_bias: expected [{hq}, 2 R + 1], got {tuple(distance_bias.shape)}")
        if distance_bias.dtype is not torch.float32 or distance_bias.get_device() != device:
            raise ValueError(f"distance_bias: expected float32 on {q.device}, got {distance_bias.dtype} on {distance_bias.device}")


def supported(q, k, v, ranges, distance_bias) -> bool:
    return (_lib.available() and q.is_cuda and q.dtype in _DTYPES and q.shape[3] in (64, 128) and ranges.plan is not None
            and q.numel() > 0 and k.numel() > 0 and q.shape[1] <= MAX_HEADS
            and (distance_bias is None or distance_bias.shape[1] <= 2 * MAX_DISTANCE + 1))


# ------------------------------------------------------------------------------------------------ native calls

_HEAD = struct.Struct("@l iiii iiii ii PPP 9l PPP PP ff")           # everything that the forward kernel reads but the status word
_TAIL = struct.Struct("@PP PPP 9l PP P")
_ARGS = struct.Struct("@l iiii iiii ii PPP 9l PPP PP ff PP PPP 9l PP P")
_NO_BACKWARD = bytes(_TAIL.size - 16)
_SCRATCH = struct.Struct("@PP")
# Up to so many keys a trained call keeps the output before rounding: dP - delta of few keys is small against either.  Relative errors of dQ and dK without
# and with it: 2 keys 3.9e-3 / 2.4e-3, 16 causal ones 2.8e-3 / 2.3e-3, 128 2.6e-3 / 2.4e-3, 512 2.5e-3 / 2.3e-3 (rounding the results alone: 1.7e-3); forward and
# backward of 8 x 128 tokens, 32 + 8 heads of 128, 40 / 45 us, of 8 x 256 67 / 83.  It goes by the length of the keys, which the host knows, not by what a query
# sees: documents of a few tokens within longer sequences keep the larger error.
WIDE_KEYS = 128
FEW_ROWS = 32           # queries of a group that the kernels for few queries take


def _rows(t):
    """Operand that the copies can address: contiguous rows at 16-byte boundaries, steps of any size above 0."""
    sb, sh, st, sd = t.stride()
    if sd == 1 and not t.data_ptr() & 15 and not (sb | sh | st) & 7 and sb > 0 and sh > 0 and st > 0:
        return t
    B, H, S, _ = t.shape        # a dimension of one is never stepped over
    if sd == 1 and not t.data_ptr() & 15 and all(n == 1 or (s > 0 and not s & 7) for n, s in ((B, sb), (H, sh), (S, st))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _like(x):
    """A gradient in ``x``'s order of heads and tokens."""
    B, H, S, D = x.shape
    return x.new_empty_strided((B, H, S, D), (S * H * D, D, H * D, 1)) if x.stride(1) < x.stride(2) else x.new_empty((B, H, S, D))


def _pack(q, k, v, ranges, out, out32, lse, scale, softcap, bias):
    B, hq, n, D = q.shape
    return _HEAD.pack(_ARGS.size, B, hq, k.shape[1], n, k.shape[2], D, _DTYPES[q.dtype], -1 if bias is None else bias.shape[1] >> 1, ranges.causal, 0,
                      q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                      out.data_ptr(), 0 if out32 is None else out32.data_ptr(), lse.data_ptr(), ranges.plan.data_ptr(),
                      0 if bias is None else bias.data_ptr(), scale, softcap)


def _forward(q, k, v, ranges, scale, softcap, bias, wide):
    B, hq, n, D = q.shape
    out = q.new_empty((B, n, hq * D))
    out32 = q.new_empty((B, n, hq * D), dtype=torch.float32) if wide else None
    lse = q.new_empty((B, hq, (n + TILE - 1) // TILE * TILE), dtype=torch.float32)
    head, status = _pack(q, k, v, ranges, out, out32, lse, scale, softcap, bias) + _NO_BACKWARD, status_tensor(q.device).data_ptr()
    scratch = None
    if not wide and n * (hq // k.shape[1]) <= FEW_ROWS:
        size = _lib.lib().tt_attn_ranges_fwd_floats(head + _SCRATCH.pack(0, status))
        if size:
            scratch = q.new_empty((size,), dtype=torch.float32)
            _lib.LAUNCHES += 1          # the join
    call("tt_attn_ranges_fwd", head + _SCRATCH.pack(0 if scratch is None else scratch.data_ptr(), status), stream())
    return out, out32, lse


def _backward(ctx, dout):
    q, k, v, bias, out, lse, _ = ctx.saved_tensors
    B, hq, n, D = q.shape
    with on_device(q):
        dout = dout.contiguous()
        if dout.data_ptr() & 15:
            dout = dout.clone()
        dq, dk, dv = _like(q), _like(k), _like(v)
        delta = lse.new_empty(lse.shape)
        dbias = partials = None
        if bias is not None and ctx.needs_input_grad[3]:
            _lib.LAUNCHES += 1          # the sum of the bias's gradients
            dbias = bias.new_empty(bias.shape)
            partials = lse.new_empty((B * hq * (lse.shape[2] // TILE) * bias.shape[1],))
        call("tt_attn_ranges_bwd", _pack(q, k, v, ctx.ranges, out, out if ctx.wide else None, lse, ctx.scale, ctx.softcap, bias)
             + _TAIL.pack(dout.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *dq.stride()[:3], *dk.stride()[:3],
                          *dv.stride()[:3], 0 if dbias is None else dbias.data_ptr(), 0 if partials is None else partials.data_ptr(),
                          status_tensor(q.device).data_ptr()), stream())
    a, b, c, d = ctx.needs_input_grad[:4]
    return dq if a else None, dk if b else None, dv if c else None, dbias if d else None, None, None, None


_backward_once = once_differentiable(_backward)


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, ranges, scale, softcap):
        q, k, v = _rows(q), _rows(k), _rows(v)
        bias = None if bias is None else bias.contiguous()
        # a bias that is trained needs the output before rounding, to more than P's 16 bits (4 bytes an element, kept for the backward), and so
        # do few keys, of which dP - delta leaves little
        wide = k.shape[2] <= WIDE_KEYS or (bias is not None and ctx.needs_input_grad[3])
        out, out32, lse = _forward(q, k, v, ranges, scale, softcap, bias, wide)
        ctx.save_for_backward(q, k, v, bias, out32 if wide else out, lse, ranges.plan)
        ctx.ranges, ctx.scale, ctx.softcap, ctx.wide = ranges, scale, softcap, wide
        return out

    @staticmethod
    def backward(ctx, dout):
        # the wrapper, which a second derivative would need to fail in, costs the host 5 us of a first one
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, dout)


def masked_attention(q, k, v, ranges, scale, softcap, distance_bias):
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    softcap = 0.0 if softcap is None else float(softcap)
    with on_device(q):
        # under a forward-mode level operands may have tangents, which the autograd function refuses and a kernel alone would lose
        if forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, distance_bias))):
            return _MaskedAttention.apply(q, k, v, distance_bias, ranges, scale, softcap)
        bias = None if distance_bias is None else distance_bias.contiguous()
        return _forward(_rows(q), _rows(k), _rows(v), ranges, scale, softcap, bias, False)[0]
