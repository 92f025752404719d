"""Rotary positions and per-head RMS norm in 64 bits, by complex multiplication, for the tests of ``ops.rotary`` and ``ops.qk_norm_rotary``."""



import torch


def angles(positions, inv_freq, axis=None):
    """``[B or 1, tokens, pairs]`` radians from ``positions [B or 1, axes, tokens]``."""
    p = positions.double()
    per_pair = torch.stack([p[:, 0 if axis is None else int(axis[j])] * float(inv_freq[j]) for j in range(len(inv_freq))], dim=-1)
    return per_pair


def turn(x, angle, amplitude, interleaved):
    """``x [B, h, S, D]`` (64 bits), its first ``2 * pairs`` elements rotated."""
    P = angle.shape[-1]
    z = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]
    head, rest = x[..., :2 * P], x[..., 2 * P:]
    if interleaved:
        pairs = torch.complex(head[..., 0::2].contiguous(), head[..., 1::2].contiguous()) * z
        out = torch.view_as_real(pairs).flatten(-2)
    else:
        pairs = torch.complex(head[..., :P].contiguous(), head[..., P:].contiguous()) * z
        out = torch.cat([pairs.real, pairs.imag], dim=-1)
    return torch.cat([out, rest], dim=-1)


def pair_size(x, P, amplitude, interleaved):
    """What a rotation's rounding errors scale with: the sum of a pair's absolute values at both of its places."""
    a = x.abs()
    head, rest = a[..., :2 * P], a[..., 2 * P:]
    if interleaved:
        s = (head[..., 0::2] + head[..., 1::2]).repeat_interleave(2, dim=-1)
    else:
        s = (head[..., :P] + head[..., P:]).repeat(1, 1, 1, 2)
    return torch.cat([amplitude * s, rest], dim=-1)


def inverse_frequencies(dim, theta):
    return [theta ** (-2.0 * j / dim) for j in range(dim // 2)]


def rounding(dtype, want):
    """Half a step of ``dtype`` at ``want``: eps / 2 of the value, and of the smallest normal number below it (fp16 is spaced 2^-24
    below 2^-14, so a value there rounds by up to 2^-25 = 2^-14 * 2^-11 however small it is)."""
    f = torch.finfo(dtype)
    return f.eps / 2 * want.abs().clamp_min(f.smallest_normal)


U32 = 2.0 ** -24
# One rotated element in fp32: the angle's part of a turn rounded (pi 2^-25), cos and sin (2 units in the last place each) times the
# amplitude, two products and a sum: below 16 roundings of a pair's size.
ROTATION = 16 * U32


def norm_error(D):
    """Relative error of ``x rsqrt(mean x^2 + eps) w`` in fp32: a sum of D squares in any order, halved by the root, and a few products."""
    return (D / 2 + 16) * U32


def close(got, want, bound, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((err - bound).max())} at {int((err - bound).argmax())}"


