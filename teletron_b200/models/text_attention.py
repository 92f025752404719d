"""The text encoders' self-attention on this package's operators instead of their library's.

:func:`use_native_attention` exchanges the attention modules of an installed ``LlamaModel`` or ``T5EncoderModel`` for ones that keep their
weights and call :mod:`teletron_b200.ops`: rotation by half layout with the configuration's scaling and causal masked attention with
shared key heads (``llama``), masked attention with the learned bias of the distance (``t5``).  The reference runs both encoders through that
library (``teletron/models/hunyuanvideo/text_encoder.py:125-238``).
"""

from __future__ import annotations

import math
import threading
from typing import NamedTuple, Optional

import torch
from torch import nn

from .. import ops


def distance_buckets(max_distance: int, num_buckets: int, bidirectional: bool = True, device=None) -> torch.Tensor:
    """Bucket of every distance ``-max_distance .. max_distance`` (key position - query position): half of a side's buckets hold one
    distance each, the others grow with its logarithm up to ``max_distance``, from where on all share the last."""
    d = torch.arange(-max_distance, max_distance + 1, device=device)
    out = torch.zeros_like(d)
    if bidirectional:
        num_buckets //= 2
        out = (d > 0).long() * num_buckets
        d = d.abs()
    else:
        d = (-d).clamp_min(0)
    exact = num_buckets // 2
    large = exact + (torch.log(d.clamp_min(1).float() / exact) / math.log(max_distance / exact) * (num_buckets - exact)).long()
    return out + torch.where(d < exact, d, large.clamp_max(num_buckets - 1))


def prompt_ranges(mask: Optional[torch.Tensor], batch: int, length: int, causal: bool, device) -> ops.KeyRanges:
    """Runs of keys for prompts that are padded on one side; ``mask [batch, length]`` on the host (it comes from the tokenizer)."""
    if mask is None or bool(mask.bool().all()):
        return ops.key_ranges(length, batch=batch, causal=causal, device=device)
    mask = mask.bool().cpu()
    n = mask.sum(dim=1)
    at = torch.arange(length)
    if torch.equal(mask, at < n[:, None]):          # padded tokens see the prompt, as in the library; nobody sees them
        return ops.key_ranges(length, batch=batch, causal=causal, kv_valid_len=n, device=device)
    if torch.equal(mask, at >= length - n[:, None]):
        return ops.key_ranges(length, batch=batch, causal=causal, documents=torch.stack([length - n, torch.full_like(n, length)], dim=1), device=device)
    raise ValueError("native attention takes prompts that are padded on one side")


class _Prepared(NamedTuple):
    """What the layers of one call share."""
    ranges: ops.KeyRanges
    positions: Optional[torch.Tensor] = None
    freqs: Optional[ops.Rotary] = None
    bias: Optional[torch.Tensor] = None


class _Shared:
    """The prepared call of every thread, so that threads on one model do not see one another's masks."""

    def __init__(self):
        self._mine, self._last, self._threads = threading.local(), None, set()

    def prepare(self, **call) -> None:
        self._mine.call = self._last = _Prepared(**call)
        self._threads.add(threading.get_ident())

    def call(self) -> _Prepared:
        call = getattr(self._mine, "call", None)
        if call is None and len(self._threads) == 1:        # another thread goes on with it: autograd's, which computes checkpointed layers again
            call = self._last
        if call is None:
            raise ValueError("native attention: prepare(...) has to be called ahead of the model, by the same thread")
        return call

    def __reduce__(self):       # a copy begins unprepared
        return _Shared, ()


class LlamaSelfAttention(nn.Module):
    def __init__(self, inner: nn.Module, shared: _Shared):
        super().__init__()
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = inner.q_proj, inner.k_proj, inner.v_proj, inner.o_proj
        self.head_dim, self.scaling = inner.head_dim, inner.scaling
        self.shared = shared

    def forward(self, hidden_states, **_):
        B, L, _ = hidden_states.shape
        q, k, v = (p(hidden_states).view(B, L, -1, self.head_dim).transpose(1, 2) for p in (self.q_proj, self.k_proj, self.v_proj))
        call = self.shared.call()
        q, k = ops.rotary(q, k, call.positions, call.freqs)
        return self.o_proj(ops.masked_attention(q, k, v, call.ranges, scale=self.scaling)), None


class T5SelfAttention(nn.Module):
    def __init__(self, inner: nn.Module, shared: _Shared):
        super().__init__()
        self.q, self.k, self.v, self.o = inner.q, inner.k, inner.v, inner.o
        if inner.has_relative_attention_bias:
            self.relative_attention_bias = inner.relative_attention_bias
        self.head_dim, self.shared = inner.key_value_proj_dim, shared

    def forward(self, hidden_states, **_):
        B, L, _ = hidden_states.shape
        q, k, v = (p(hidden_states).view(B, L, -1, self.head_dim).transpose(1, 2) for p in (self.q, self.k, self.v))
        call = self.shared.call()
        o = ops.masked_attention(q, k, v, call.ranges, scale=1.0, distance_bias=call.bias)
        return self.o(o.to(self.o.weight.dtype)), None


def rotary_of(cfg) -> ops.Rotary:
    """Frequencies of a model configuration.  Releases ahead of 5 of the encoders' package keep the scaling in ``rope_scaling`` and the rest beside it."""
    rope = getattr(cfg, "rope_parameters", None)
    rope = dict((getattr(cfg, "rope_scaling", None) if rope is None else rope) or {})
    head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
    part = rope.get("partial_rotary_factor") or getattr(cfg, "partial_rotary_factor", None) or 1.0
    theta = rope.get("rope_theta") or getattr(cfg, "rope_theta", None) or 10000.0
    return ops.rotary_frequencies(int(head_dim * part), float(theta), scaling=rope)


def _check_rotary(model, freqs: ops.Rotary) -> None:
    """Raises ``ValueError`` where the model's own table says otherwise (16-bit models hold it in 16 bits)."""
    own = getattr(model, "rotary_emb", None)
    inv = getattr(own, "inv_freq", None)
    if inv is None or inv.is_meta:
        return
    amplitude = getattr(own, "attention_scaling", freqs.amplitude)
    if inv.shape != freqs.inv_freq.shape or not torch.allclose(inv.double().cpu(), freqs.inv_freq, rtol=2 ** -7, atol=2 ** -24) \
            or not math.isclose(amplitude, freqs.amplitude, rel_tol=2 ** -7):
        raise ValueError("native attention: the model rotates by other frequencies than its configuration says")


class _NativeLlama:
    def __init__(self, model):
        self.shared, self.freqs = _Shared(), rotary_of(model.config)
        _check_rotary(model, self.freqs)
        self.freqs = self.freqs.to(model.embed_tokens.weight.device)
        for layer in model.layers:
            layer.self_attn = LlamaSelfAttention(layer.self_attn, self.shared)

    def prepare(self, mask, batch, length, device):
        self.freqs = freqs = self.freqs.to(device)          # the model may have moved
        self.shared.prepare(ranges=prompt_ranges(mask, batch, length, True, device), freqs=freqs,
                            positions=torch.arange(length, device=device, dtype=torch.int32))


class _NativeT5:
    def __init__(self, model):
        self.shared, cfg = _Shared(), model.config
        for block in model.encoder.block:
            block.layer[0].SelfAttention = T5SelfAttention(block.layer[0].SelfAttention, self.shared)
        self.table = model.encoder.block[0].layer[0].SelfAttention.relative_attention_bias
        self.buckets = distance_buckets(cfg.relative_attention_max_distance, cfg.relative_attention_num_buckets, device=self.table.weight.device)

    def prepare(self, mask, batch, length, device):
        self.shared.prepare(ranges=prompt_ranges(mask, batch, length, False, device), bias=self.table.weight[self.buckets].t().float().contiguous())


def use_native_attention(model):
    """Exchanges the attention modules of a ``LlamaModel`` or ``T5EncoderModel`` in place.  Returns an object whose
    ``prepare(mask, batch, length, device)`` has to be called ahead of each call of the model, by the same thread, with the tokenizer's mask or
    None."""
    kind = type(model).__name__
    if kind == "LlamaModel":
        return _NativeLlama(model)
    if kind == "T5EncoderModel":
        return _NativeT5(model)
    raise ValueError(f"native attention is there for LlamaModel and T5EncoderModel, not for {kind}")
