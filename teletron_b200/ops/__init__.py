"""Functional op layer.

Every op has two implementations behind one signature:

* ``reference`` - pure PyTorch (CPU capable, plain autograd); the numerics oracle and
  the restated library baseline.
* ``cuda`` - hand-written sm_100a kernels from ``teletron_b200/csrc`` reached through
  ``ctypes`` (:mod:`teletron_b200.ops._lib`), wrapped in ``autograd.Function``s.

Selection: :func:`set_impl` (``"auto" | "torch" | "cuda"``).  ``auto`` uses the CUDA
kernels for CUDA bf16 tensors and the reference otherwise.  On a machine with a GPU the
native library must be present: there is no silent fallback (set
``TELETRON_B200_ALLOW_FALLBACK=1`` to opt into one, e.g. for the baseline arm).
"""

from __future__ import annotations

import contextlib
import os

import torch

from . import reference
from . import attn_ranges
from . import rope
from . import optim  # noqa: F401
from .attn_ranges import KeyRanges, key_ranges  # noqa: F401
from .rope import Rotary, rotary_frequencies  # noqa: F401

_IMPL = os.environ.get("TELETRON_B200_IMPL", "auto")


def set_impl(name: str) -> None:
    global _IMPL
    if name not in ("auto", "torch", "cuda"):
        raise ValueError(name)
    _IMPL = name


def get_impl() -> str:
    return _IMPL


_NVTX = os.environ.get("TELETRON_B200_NVTX", "0") == "1"


def set_nvtx(enabled: bool) -> None:
    """Named ranges around blocks and steps for a timeline profiler (set by ``--profile``)."""
    global _NVTX
    _NVTX = bool(enabled)


@contextlib.contextmanager
def nvtx_range(name: str):
    """``torch.cuda.nvtx`` range when enabled and CUDA is present; otherwise free."""
    if _NVTX and torch.cuda.is_available():
        torch.cuda.nvtx.range_push(name)
        try:
            yield
        finally:
            torch.cuda.nvtx.range_pop()
    else:
        yield


@contextlib.contextmanager
def impl(name: str):
    prev = get_impl()
    set_impl(name)
    try:
        yield
    finally:
        set_impl(prev)


def _use_cuda(*tensors: torch.Tensor, dtypes=(torch.bfloat16,)) -> bool:
    """True when the sm_100a kernels should run for these operands (``dtypes``: the types that the op's kernels take)."""
    if _IMPL == "torch":
        return False
    t0 = tensors[0]
    if not t0.is_cuda:
        if _IMPL == "cuda":
            raise RuntimeError("impl='cuda' requested for a non-CUDA tensor")
        return False
    if t0.dtype not in dtypes:
        if _IMPL == "cuda":
            raise RuntimeError("the sm_100a kernels take %s operands, got %s"
                               % (" / ".join({"bfloat16": "bf16", "float16": "fp16", "float32": "fp32"}[str(d)[6:]] for d in dtypes), t0.dtype))
        return False
    from . import _lib
    if not _lib.available():
        if os.environ.get("TELETRON_B200_ALLOW_FALLBACK") == "1" and _IMPL != "cuda":
            return False
        raise RuntimeError(
            "teletron_b200 native library is not built (run `python -m teletron_b200.build`); "
            "refusing to fall back to library kernels on a GPU: " + _lib.load_error())
    return True


def layernorm_modulate(x, scale, shift, eps: float = 1e-6):
    if _use_cuda(x):
        from . import cuda_ops
        return cuda_ops.layernorm_modulate(x, scale, shift, eps)
    return reference.layernorm_modulate(x, scale, shift, eps)


def gate_residual(residual, branch, gate):
    if _use_cuda(residual):
        from . import cuda_ops
        return cuda_ops.gate_residual(residual, branch, gate)
    return reference.gate_residual(residual, branch, gate)


def gate_residual_layernorm_modulate(residual, branch, gate, scale, shift, eps: float = 1e-6):
    if _use_cuda(residual):
        from . import cuda_ops
        return cuda_ops.gate_residual_layernorm_modulate(residual, branch, gate, scale, shift, eps)
    return reference.gate_residual_layernorm_modulate(residual, branch, gate, scale, shift, eps)


def rmsnorm(x, weight, eps: float = 1e-6):
    if _use_cuda(x):
        from . import cuda_ops
        return cuda_ops.rmsnorm(x, weight, eps)
    return reference.rmsnorm(x, weight, eps)


def apply_rope(x, cos, sin):
    return reference.apply_rope(x, cos, sin)


_ROTARY_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _rotary_kernel_ok(q) -> bool:
    if not _use_cuda(q, dtypes=_ROTARY_DTYPES):
        return False
    if rope.supported(q):
        return True
    from . import fallback
    fallback.note("rotary", f"q {tuple(q.shape)} {q.dtype}")
    return False


def rotary(q, k, positions, freqs):
    """Queries and keys ``[batch, heads, tokens, head_dim]`` (any strides, head counts of their own) rotated by their positions.

    ``positions``: int32 or int64, ``[tokens]`` or ``[batch, tokens]``, with several axes ``[axes, tokens]`` or ``[batch, axes, tokens]``;
    ``freqs``: what :func:`rotary_frequencies` returns.  ``k`` may be None.  Returns head-major ``(q, k)`` of the same type; the gradients
    come in the order of the inputs.  bf16, fp16 and fp32."""
    stride = rope.check_arguments(q, k, positions, freqs)
    if _rotary_kernel_ok(q):
        return rope.rotary(q, k, positions, stride, freqs)
    return reference.rotary(q, k, rope.by_axis(positions, freqs.num_axes), freqs)


def qk_norm_rotary(q, k, q_weight, k_weight, positions, freqs, eps: float = 1e-6):
    """RMS norm of every head of ``q`` and ``k`` (weights ``[head_dim]``, statistics in fp32), then :func:`rotary`, rounded once."""
    stride = rope.check_arguments(q, k, positions, freqs)
    rope.check_norm(q, k, q_weight, k_weight, eps)
    if _rotary_kernel_ok(q):
        return rope.qk_norm_rotary(q, k, q_weight, k_weight, positions, stride, freqs, eps)
    return reference.qk_norm_rotary(q, k, q_weight, k_weight, rope.by_axis(positions, freqs.num_axes), freqs, eps)


def linear(x, weight, bias=None, activation=None):
    if _use_cuda(x):
        from . import cuda_ops
        return cuda_ops.linear(x, weight, bias, activation)
    return reference.linear(x, weight, bias, activation)


def linear_merged(x1, x2, weight, bias=None):
    """``cat([x1, x2], -1) @ weight^T + bias`` without ever forming the concatenated gradient in the backward."""
    if _use_cuda(x1):
        from . import cuda_ops
        return cuda_ops.linear_merged(x1, x2, weight, bias)
    return reference.linear_merged(x1, x2, weight, bias)


def attention(q, k, v, kv_valid_len=None, scale=None, mask_range=None):
    """``kv_valid_len`` masks the key tail, ``mask_range = (lo, hi)`` one more key range."""
    if _use_cuda(q):
        from . import cuda_ops
        return cuda_ops.attention(q, k, v, kv_valid_len, scale, mask_range)
    return reference.attention(q, k, v, kv_valid_len, scale, mask_range)


def masked_attention(q, k, v, ranges, scale=None, softcap=None, distance_bias=None):
    """Softmax attention in which every query sees one run of the keys: causal, prefix and document masks, padded batches, caches.

    ``q [batch, heads, queries, head_dim]``, ``k``, ``v`` ``[batch, key heads, keys, head_dim]`` (any strides; the heads are a multiple of the key
    heads); ``ranges``: what :func:`key_ranges` returns.  ``scale`` defaults to ``head_dim ** -0.5``; ``softcap`` caps the scaled scores as
    ``softcap * tanh(s / softcap)``; ``distance_bias [heads, 2 R + 1]`` (fp32) is added for the distance key position - query position, distances
    beyond R taking the ends' values.  Returns token-major ``[batch, queries, heads * head_dim]``, 0 for queries that see nothing.

    Keys, values, queries and output gradients that no run reaches (padding) may hold anything; those that some query sees have to be finite,
    as a query's weights of 0 still multiply what its neighbours see.  Kernels: bf16 and fp16, head_dim 64 and 128, R up to 1024."""
    attn_ranges.check_arguments(q, k, v, ranges, scale, softcap, distance_bias)
    if _use_cuda(q, dtypes=(torch.bfloat16, torch.float16)):
        if attn_ranges.supported(q, k, v, ranges, distance_bias):
            return attn_ranges.masked_attention(q, k, v, ranges, scale, softcap, distance_bias)
        if q.numel() and k.numel():             # nothing to compute is no fallback
            from . import fallback
            fallback.note("masked_attention", f"q {tuple(q.shape)} {q.dtype}")
    return reference.masked_attention(q, k, v, ranges, scale, softcap, distance_bias)


def qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin, num_heads,
                   eps: float = 1e-6, rope_len=None):
    if _use_cuda(x):
        from . import cuda_ops
        return cuda_ops.qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin,
                                       num_heads, eps, rope_len)
    return reference.qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin,
                                    num_heads, eps, rope_len)


def joint_qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin, x2, weight2, bias2,
                         q_norm_weight2, k_norm_weight2, num_heads, eps: float = 1e-6):
    """Video stream ``x`` (RoPE applied) and text stream ``x2`` (no RoPE), each with its own weights,
    projected into shared ``[B, heads, S + T, D]`` q / k / v (video tokens first)."""
    if _use_cuda(x) and q_norm_weight.shape[0] == 128:
        from . import cuda_ops
        return cuda_ops.joint_qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin, x2, weight2,
                                             bias2, q_norm_weight2, k_norm_weight2, num_heads, eps)
    return reference.joint_qkv_projection(x, weight, bias, q_norm_weight, k_norm_weight, cos, sin, x2, weight2,
                                          bias2, q_norm_weight2, k_norm_weight2, num_heads, eps)


def _flow_kernel_ok(*tensors) -> bool:
    t0 = tensors[0]
    return (t0.is_cuda and all(t.dtype == torch.bfloat16 and t.shape == t0.shape for t in tensors)
            and (t0.numel() // max(1, t0.shape[0])) % 8 == 0 and _use_cuda(t0))


def flow_match_loss(pred, noise, latents, weight):
    if _flow_kernel_ok(pred, noise, latents):
        from . import cuda_ops
        return cuda_ops.flow_match_loss(pred, noise, latents, weight)
    return reference.flow_match_loss(pred, noise, latents, weight)


def noise_mix(latents, noise, sigma):
    """Model input of a flow-matching step: ``(1 - sigma) * latents + sigma * noise`` with one noise level per sample."""
    if _flow_kernel_ok(latents, noise):
        from . import cuda_ops
        return cuda_ops.noise_mix(latents, noise, sigma)
    return reference.noise_mix(latents, noise, sigma)
