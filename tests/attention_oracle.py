"""Attention over runs of keys in 64 bits from its definition, with the sizes that rounding errors scale with, for the tests of ``ops.masked_attention``."""

import math

import torch

U16 = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step of a 16-bit type, relative


def runs(q_len, kv_len, batch, causal=False, documents=None, prefix=0, kv_valid=None, start=0):
    """First and behind-last key of every query by going through the definition, ``[batch, q_len]`` lists."""
    first, behind = torch.zeros(batch, q_len, dtype=torch.int32), torch.zeros(batch, q_len, dtype=torch.int32)
    for b in range(batch):
        off = None if documents is None else documents[b] if isinstance(documents[0], list) else documents
        length = kv_len if kv_valid is None else kv_valid[b] if isinstance(kv_valid, list) else kv_valid
        at = start[b] if isinstance(start, list) else start
        for i in range(q_len):
            seen = []
            for j in range(min(kv_len, length)):
                doc, origin = 0, 0
                if off is not None:
                    mine = [d for d in range(len(off) - 1) if off[d] <= i < off[d + 1]]
                    if not mine or not (off[mine[0]] <= j < off[mine[0] + 1]):
                        continue
                    doc, origin = mine[0], off[mine[0]]
                p = prefix
                if isinstance(p, list):
                    p = p[b][doc] if isinstance(p[b], list) else p[b]
                if causal and j > at + i and j - origin >= p:
                    continue
                seen.append(j)
            if seen:
                assert seen == list(range(seen[0], seen[-1] + 1))
                first[b, i], behind[b, i] = seen[0], seen[-1] + 1
    return first, behind


U32 = 2.0 ** -24                                                  # half a step of fp32, relative


def rounding(dtype, want):
    """Half a step at ``want``, which below the smallest normal number no longer shrinks."""
    f = torch.finfo(dtype)
    return f.eps / 2 * want.abs().clamp_min(f.smallest_normal)


def attention(q, k, v, first, behind, scale, dtype, softcap=None, bias=None, start=None, dout=None):
    """Values in 64 bits, head-major, and bounds of what the kernels may be off by: ``{name: (value, bound)}`` of ``out`` and, with
    ``dout [B, h, n, D]``, ``dq``, ``dk``, ``dv``, ``dbias``.

    The bounds follow the roundings.  u = 2^-24 for sums and functions in 32 bits (a product over n terms: n + 8 of them, twice for the tensor core's
    truncation), U for half a step of the 16-bit type, t its absolute floor (2^-25 in fp16, whose numbers below 2^-14 are evenly spaced; P and dS
    are of the order of 1 there).
      score      (2 D + 16) u sum |q||k| |scale|, behind the cap times its slope, 8 u of the cap, 4 u of |bias| and of |s|
      P          score errors of the key and of the row's maximum (in the sum), 2 n u of the sum: rel.  Rounded to 16 bits: U + t
      out        sum (P (U + rel) + t) |v|, and its rounding
      dS         P's error times |dP - delta|, P times the errors of dP ((2 D + 16) u sum |dO||v|) and delta (sum |dO| out's error)
      dS'        the slope in fp16 (2^-11, 2^-24), the rounding U + t
      dQ, dK, dV their sums' 2 n u, and their rounding;   dbias: dS's error with P unrounded and out to 2 U^2, sums of n m B terms"""
    U, u, t = U16[dtype], U32, 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133
    q, k, v = q.double(), k.double(), v.double()
    B, h, n, D = q.shape
    G, m = h // k.shape[1], k.shape[2]
    j = torch.arange(m, device=q.device)
    see = ((j >= first[..., None]) & (j < behind[..., None]))[:, None]            # [B, 1, n, m]
    used, live = see.any(2)[..., None], see.any(3)[..., None]                    # [B, 1, m, 1], [B, 1, n, 1]
    q = q.masked_fill(~live, 0.0)
    k, v = (x.masked_fill(~used, 0.0).repeat_interleave(G, 1) for x in (k, v))
    raw = (q @ k.mT) * scale
    s, slope = raw, torch.ones_like(raw)
    if softcap:
        th = torch.tanh(raw / softcap)
        s, slope = softcap * th, 1 - th * th
    score = (2 * D + 16) * u * abs(scale) * (q.abs() @ k.abs().mT) * slope + (8 * u * softcap if softcap else 0.0)
    far = None
    if bias is not None:
        R = (bias.shape[1] - 1) // 2
        i = torch.arange(n, device=q.device).expand(B, n) + (0 if start is None else start[:, None].long())
        far = (j - i[..., None]).clamp(-R, R) + R                                # [B, n, m]
        add = bias.double()[:, far].transpose(0, 1)
        s, score = s + add, score + 4 * u * add.abs().nan_to_num(posinf=0.0)
    score = torch.where(see, score + 4 * u * s.abs().nan_to_num(posinf=0.0), torch.zeros_like(score))
    s = torch.where(see, s, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(s.amax(-1, keepdim=True) > -math.inf, p, torch.zeros_like(p))
    rel = score + score.amax(-1, keepdim=True) + (2 * m + 32) * u
    out = p @ v
    p_err = p * (U + rel) + t * see
    out_err = p_err @ v.abs() + 2 * m * u * (p @ v.abs())
    res = dict(out=(out, out_err + rounding(dtype, out)))
    if dout is None:
        return res
    do = dout.double().masked_fill(~live, 0.0)
    dp, size = do @ v.mT, do.abs() @ v.abs().mT
    delta = (do * out).sum(-1, keepdim=True)
    ds0 = p * (dp - delta)
    dp_err = (2 * D + 16) * u * size
    delta_err = (do.abs() * res["out"][1]).sum(-1, keepdim=True) + (D + 8) * u * (do * out).abs().sum(-1, keepdim=True)
    ds0_err = p_err * ((dp - delta).abs() + dp_err + delta_err) + p * (dp_err + delta_err)
    ds = ds0 * slope
    ds_err = ds0_err * slope + (ds0.abs() + ds0_err) * (2.0 ** -11 * slope + 2.0 ** -24 if softcap else 0.0)
    ds_err = ds_err + U * (ds.abs() + ds_err) + t * see
    join = lambda x: x.view(B, h // G, G, m, D).sum(2)

    def product(a, a_err, b, wrap, factor=1.0):
        value = factor * wrap(a @ b)
        return value, wrap(abs(factor) * (a_err @ b.abs() + 2 * (a.shape[-1] * G + 8) * u * (a.abs() @ b.abs()))) + rounding(dtype, value)

    res["dq"] = product(ds, ds_err, k, lambda x: x, scale)
    res["dk"] = product(ds.mT, ds_err.mT, q, join, scale)
    res["dv"] = product(p.mT, p_err.mT, do, join)
    if bias is not None:
        wide = p * (2 * U * U + rel) + t * t * see
        delta_err = (do.abs() * (wide @ v.abs() + 4 * m * u * (p @ v.abs()))).sum(-1, keepdim=True) + (D + 8) * u * (do * out).abs().sum(-1, keepdim=True)
        err = p * rel * (dp - delta).abs() + p * (dp_err + delta_err) + (n + m + 64 + B * n / 128) * u * ds0.abs()
        sums = []
        for x in (ds0, err):
            table = torch.zeros(h, bias.shape[1], dtype=torch.float64, device=q.device)
            for b in range(B):
                for hh in range(h):
                    table[hh].index_add_(0, far[b].flatten(), x[b, hh].flatten())
            sums.append(table)
        res["dbias"] = tuple(sums)
    return res


def close(got, pair, what=""):
    want, bound = pair
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((err - bound).nan_to_num(1e30).max())}"
