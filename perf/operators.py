"""The operators between a projection and an attention layer's output, as a list of measurable cases.

* ``rotary``: queries and keys rotated by their positions (``ops.rotary``): interleaved and half layouts, part of the
  head, several position axes, frequencies scaled for long contexts.
* ``norm_rotary``: the same behind an RMS norm of every head of the queries and keys (``ops.qk_norm_rotary``).
* ``attention``: softmax attention in which every query sees one run of the keys (``ops.masked_attention`` over
  ``ops.key_ranges``): causal, prefix and document masks, caches, shared key heads, scores capped by a tanh, a bias that
  depends on the distance.

Head counts, widths and lengths are those of the text encoders (32 query and 8 key heads of 128 with 8192 positions; 64
heads of 64; prompts of 256 tokens) and of the 13B video model (24 heads of 128; 720P x 33 frames are 9 x 45 x 80 video
tokens, 32656 with the prompt).  Where :data:`own` is false, ``run`` computes the same from elementary torch operations in 32
bits.  ``exact`` gives the values in 64 bits, from the definitions.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases

def _rotary(name, op="rotary", **kw):
    case = dict(name=name, op=op, batch=1, tokens=1, frames=0, rows=0, columns=0, q_heads=32, k_heads=8, head_dim=128, rotary_dim=128,
                layout="half", scaling="none", theta=10000.0, start=0, packed=True, dtype="bf16", train=False)
    case.update(kw)
    return case


def _attention(name, **kw):
    case = dict(name=name, op="attention", batch=1, queries=1, keys=1, q_heads=32, k_heads=8, head_dim=128, causal=False, documents=0,
                prefix=0, cache=False, softcap=0.0, distances=0, layout="token", dtype="bf16", train=False)
    case.update(kw)
    return case


def listed():
    return [
        # one new token for each of eight requests, far into their contexts: launch latency
        _rotary("rotary_token", batch=8, start=7000, scaling="llama3", theta=500000.0),
        # a text encoder's longest batch, in the type it runs in by default
        _rotary("rotary_text_8192", batch=4, tokens=8192, theta=500000.0, scaling="llama3", dtype="fp16"),
        # the video stream's three axes (16 + 56 + 56 of 128), a training step of one block at 720P x 33 frames
        _rotary("rotary_video_train", tokens=32400, frames=9, rows=45, columns=80, k_heads=24, q_heads=24, layout="interleaved",
                theta=256.0, packed=False, train=True),
        # a quarter of a narrow head rotated, a length that nothing divides, frequencies stretched for long contexts, fp32
        _rotary("rotary_part_train", batch=3, tokens=1537, q_heads=12, k_heads=12, head_dim=80, rotary_dim=20, scaling="yarn",
                dtype="fp32", train=True),
        # one new token for each of 64 requests, heads normed first
        _rotary("norm_rotary_token", "norm_rotary", batch=64, start=3000),
        # QK-norm and the video stream's rotation, forward and backward, at 720P x 33 frames
        _rotary("norm_rotary_video_train", "norm_rotary", tokens=32400, frames=9, rows=45, columns=80, k_heads=24, q_heads=24,
                layout="interleaved", theta=256.0, train=True),
        # shared key heads of 64, odd length, fp16, forward and backward
        _rotary("norm_rotary_shared_train", "norm_rotary", batch=3, tokens=1001, k_heads=4, head_dim=64, rotary_dim=64, dtype="fp16",
                scaling="linear", train=True),
        # the prompt encoder: eight prompts padded to 256 tokens, causal
        _attention("attention_prompts", batch=8, queries=256, keys=256, causal=True, documents=1, dtype="fp16"),
        # an encoder with a learned bias over distances up to 128, trained: heads of 64 with a key head each
        _attention("attention_distance_train", batch=4, queries=512, keys=512, q_heads=64, k_heads=64, head_dim=64, documents=1,
                   distances=128, train=True),
        # clips of several lengths packed into one sequence of 720P x 33 frames' length, each seeing itself, trained
        _attention("attention_clips_train", queries=32656, keys=32656, q_heads=24, k_heads=24, documents=5, layout="head", train=True),
        # prompts read both ways and answered causally, capped scores, trained; an odd length
        _attention("attention_prefix_cap_train", batch=2, queries=4095, keys=4095, causal=True, prefix=611, softcap=50.0, train=True),
        # one new token for each of eight requests over caches of up to 8192 tokens
        _attention("attention_token", batch=8, queries=1, keys=8192, causal=True, cache=True, layout="head"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.55:
        op = rng.choice(["rotary", "norm_rotary"])
        head_dim = rng.choice([64, 128, 128, 80, 96, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4])
        k_heads = rng.choice([1, 2, 4, 8, 12, 24])
        q_heads = k_heads * (rng.choice([1, 1, 2, 4, 8]) if k_heads <= 8 else 1)
        video = rng.random() < 0.25
        frames, rows, columns = rng.randint(1, 9), rng.randint(2, 45), rng.randint(2, 80)
        most = max(1, 32400 * 48 * 128 // ((q_heads + k_heads) * head_dim))
        batch = 1 if video else _log_int(rng, 1, 16)
        if video:
            while frames * rows * columns > most:
                frames, rows = max(1, frames // 2), max(2, rows // 2)
                columns = max(2, columns - 8)
        tokens = frames * rows * columns if video else _log_int(rng, 1, max(1, min(32400, most // batch)))
        return _rotary(None, op, batch=batch, tokens=tokens, frames=frames if video else 0, rows=rows if video else 0,
                       columns=columns if video else 0, q_heads=q_heads, k_heads=k_heads, head_dim=128 if video else head_dim,
                       rotary_dim=128 if video else rotary_dim, layout="interleaved" if video else rng.choice(["half", "interleaved"]),
                       scaling="none" if video else rng.choice(["none", "linear", "ntk", "llama3", "yarn"]),
                       theta=rng.choice([256.0, 10000.0, 500000.0]), start=0 if video else rng.choice([0, 0, _log_int(rng, 1, 100000)]),
                       packed=rng.random() < 0.6, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), train=rng.random() < 0.6)
    k_heads = rng.choice([1, 2, 8, 12, 24])
    group = rng.choice([1, 1, 2, 4, 8]) if k_heads <= 8 else 1
    head_dim = rng.choice([64, 128])
    dtype, layout = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["head", "token"])
    if rng.random() < 0.25:
        # few new tokens over a cache
        batch = _log_int(rng, 1, 32)
        keys = _log_int(rng, 16, min(65536, 2 ** 22 // (batch * k_heads)))
        return _attention(None, batch=batch, queries=min(keys, rng.choice([1, 1, 1, 2, 5])), keys=keys, q_heads=k_heads * group,
                          k_heads=k_heads, head_dim=head_dim, causal=True, cache=True, softcap=rng.choice([0.0, 0.0, 30.0]),
                          distances=rng.choice([0, 0, 128]), layout=layout, dtype=dtype)
    queries = _log_int(rng, 1, 12000)
    batch = max(1, min(_log_int(rng, 1, 8), int(24 * 12000 ** 2 / (queries ** 2 * k_heads * group))))
    while queries ** 2 * batch * k_heads * group > 24 * 12000 ** 2:
        queries = queries * 3 // 4
    causal = rng.random() < 0.5
    documents = min(rng.choice([0, 1, 1, 3, 9]), queries)
    return _attention(None, batch=batch, queries=queries, keys=queries, q_heads=k_heads * group, k_heads=k_heads, head_dim=head_dim,
                      causal=causal, documents=documents, prefix=rng.randint(1, queries) if causal and rng.random() < 0.4 else 0,
                      softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), distances=rng.choice([0, 0, 32, 128]), layout=layout, dtype=dtype,
                      train=rng.random() < 0.6)


def _offsets(case):
    """Document offsets of every sample, ``[batch][documents + 1]``: ragged lengths, and a padded tail that no document covers."""
    out = []
    for b in range(case["batch"]):
        rng = random.Random(7919 * case["queries"] + 31 * case["documents"] + b)
        n, total = case["documents"], case["queries"]
        used = max(min(n, total), total - int(rng.random() * 0.3 / n * total))
        cuts = sorted(rng.sample(range(1, used), n - 1)) if n > 1 else []
        if n > 1 and used > 64 * n:          # none much shorter than the rest
            cuts = [int(used * (i + 0.6 * rng.random() - 0.3) / n) for i in range(1, n)]
        out.append([0] + cuts + [used])
    return out


def _cache_lengths(case):
    rng = random.Random(104729 + case["keys"])
    return [max(case["queries"], case["keys"] - int(rng.random() ** 2 * 0.6 * case["keys"])) for _ in range(case["batch"])]


def _runs(case):
    """First and behind-last visible key of every query, on the host: ``[batch, queries]`` each."""
    B, n, m = case["batch"], case["queries"], case["keys"]
    i = torch.arange(n)
    first, behind = torch.zeros(B, n, dtype=torch.long), torch.full((B, n), m, dtype=torch.long)
    if case["cache"]:
        length = torch.tensor(_cache_lengths(case))[:, None]
        return first, torch.minimum(length - n + i[None] + 1, length)
    if case["documents"]:
        first, behind = first.clone(), torch.zeros_like(behind)
        for b, off in enumerate(_offsets(case)):
            for lo, hi in zip(off, off[1:]):
                first[b, lo:hi] = lo
                behind[b, lo:hi] = hi
    if case["causal"]:
        reach = torch.maximum(i[None] + 1, first + case["prefix"])
        behind = torch.minimum(behind, reach)
    return first, behind


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] != "attention":
        rows = case["batch"] * case["tokens"]
        n = rows * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        # forward: read and written; backward: the incoming gradients read and the outgoing ones written, behind a norm the input again
        passes = 2 + (0 if not case["train"] else 2 if case["op"] == "rotary" else 3)
        return {"bytes": passes * size * n + 4 * rows, "flops": (4 if case["op"] == "rotary" else 8) * n * (2 if case["train"] else 1)}
    first, behind = _runs(case)
    seen = (behind - first).clamp_min(0)
    B, D, hq, hk = case["batch"], case["head_dim"], case["q_heads"], case["k_heads"]
    nq = B * case["queries"] * hq * D
    nk = D * hk * (sum(_cache_lengths(case)) if case["cache"] else B * case["keys"])
    if case["train"]:       # forward: q k v -> out; backward: q k v out dout -> dq dk dv
        moved = (2 * nq + 2 * nk) + (3 * nq + 2 * nk) + (nq + 2 * nk)
    else:
        moved = 2 * nq + 2 * nk
    products = 7 if case["train"] else 2
    return {"bytes": size * moved, "flops": 2 * products * D * hq * int(seen.sum())}


# ------------------------------------------------------------------------------------------------ inputs

def _scaling(case):
    """How the frequencies are stretched, as a model's configuration says it."""
    return {"none": None, "linear": dict(rope_type="linear", factor=4.0), "ntk": dict(rope_type="ntk", factor=4.0),
            "llama3": dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                           original_max_position_embeddings=8192),
            "yarn": dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)}[case["scaling"]]


def _axes(case):
    return (16, 56, 56) if case["frames"] else None


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def heads(B, S, counts, D, token_major):
        """Head-major views of one token-major buffer (what a fused projection leaves), or tensors of their own."""
        if token_major:
            buf = normal(B, S, sum(counts) * D)
            parts = buf.split([c * D for c in counts], dim=-1)
            return [p.view(B, S, c, D).transpose(1, 2) for p, c in zip(parts, counts)]
        return [normal(B, c, S, D) for c in counts]

    B, D, hq, hk = case["batch"], case["head_dim"], case["q_heads"], case["k_heads"]
    if case["op"] != "attention":
        S = case["tokens"]
        # a fused projection also holds the values behind the queries and keys
        q, k = heads(B, S, (hq, hk, hk) if case["packed"] else (hq, hk), D, case["packed"])[:2]
        st = dict(q=q, k=k)
        if case["frames"]:
            grid = torch.meshgrid(*[torch.arange(n) for n in (case["frames"], case["rows"], case["columns"])], indexing="ij")
            st["positions"] = torch.stack([x.reshape(-1) for x in grid]).to(device="cuda", dtype=torch.int32)
        else:       # every request at a place of its own, the tokens of one in a row
            at = torch.randint(0, 64, (B, 1), generator=g, device="cuda") + case["start"]
            st["positions"] = (at + torch.arange(S, device="cuda")).to(torch.int32)
        if case["op"] == "norm_rotary":
            st["q_weight"] = (1 + 0.1 * normal(D, dtype=torch.float32)).to(dt)
            st["k_weight"] = (1 + 0.1 * normal(D, dtype=torch.float32)).to(dt)
        if case["train"]:
            st["gq"], st["gk"] = normal(B, hq, S, D), normal(B, hk, S, D)
        return st
    token = case["layout"] == "token"
    if case["queries"] == case["keys"] and not case["cache"]:
        q, k, v = heads(B, case["queries"], (hq, hk, hk), D, token)
    else:
        q, = heads(B, case["queries"], (hq,), D, token)
        k, v = heads(B, case["keys"], (hk, hk), D, token)
    st = dict(q=q, k=k, v=v)
    if case["documents"]:
        st["offsets"] = torch.tensor(_offsets(case), device="cuda", dtype=torch.int32)
    if case["cache"]:
        st["lengths"] = torch.tensor(_cache_lengths(case), device="cuda", dtype=torch.int32)
    if case["distances"]:
        st["bias"] = 0.5 * normal(hq, 2 * case["distances"] + 1, dtype=torch.float32)
    if case["train"]:
        st["gout"] = normal(B, case["queries"], hq * D)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if not own:
        if case["op"] == "attention":
            st["cuts"] = _offsets(case) if case["documents"] else None
        else:
            st["inverse"], st["amplitude"] = _inverse_frequencies(case)
        return st
    from teletron_b200 import ops
    if case["op"] != "attention":
        st["rotary"] = ops.rotary_frequencies(case["rotary_dim"], case["theta"], axes=_axes(case), scaling=_scaling(case),
                                              interleaved=case["layout"] == "interleaved", device="cuda")
        leaves = ["q", "k"] + (["q_weight", "k_weight"] if case["op"] == "norm_rotary" else [])
    else:
        # the plan of a batch, which all layers share
        kw = dict(batch=case["batch"], causal=case["causal"], device="cuda")
        if case["cache"]:
            kw.update(kv_valid_len=st["lengths"], query_start=st["lengths"] - case["queries"])
        if case["documents"]:
            kw.update(documents=st["offsets"])
        if case["prefix"]:
            kw.update(prefix_len=case["prefix"])
        st["ranges"] = ops.key_ranges(case["queries"], case["keys"], **kw)
        leaves = ["q", "k", "v"] + (["bias"] if case["distances"] else [])
    if case["train"]:
        for n in leaves:
            st[n] = st[n].requires_grad_()
    st["leaves"] = leaves
    return st


def run(state):
    case = state["case"]
    if not own:
        return _plain_attention(state) if case["op"] == "attention" else _plain_rotary(state)
    from teletron_b200 import ops
    if case["op"] == "attention":
        out = ops.masked_attention(state["q"], state["k"], state["v"], state["ranges"], softcap=case["softcap"] or None,
                                   distance_bias=state.get("bias"), scale=1.0 / 8 if case["distances"] else None)
        outs, grads = {"out": out}, [state.get("gout")]
    else:
        if case["op"] == "rotary":
            q, k = ops.rotary(state["q"], state["k"], state["positions"], state["rotary"])
        else:
            q, k = ops.qk_norm_rotary(state["q"], state["k"], state["q_weight"], state["k_weight"], state["positions"], state["rotary"])
        outs, grads = {"q": q, "k": k}, [state.get("gq"), state.get("gk")]
    if case["train"]:
        leaves = state["leaves"]
        got = torch.autograd.grad(list(outs.values()), [state[n] for n in leaves], grads)
        outs = {n: t.detach() for n, t in outs.items()}
        outs.update({"d" + n: t for n, t in zip(leaves, got)})
    return outs


# ------------------------------------------------------------------------------------------------ plain forms: rotation

def _inverse_frequencies(case):
    """Radians per position of every rotated pair in 64 bits, with the axis of each (``[pairs]`` both), and the amplitude."""
    theta, scaling = case["theta"], _scaling(case) or {}
    kind = scaling.get("rope_type")
    amplitude = 1.0
    per_axis = _axes(case) or (case["rotary_dim"],)
    inverse, axis = [], []
    for a, dim in enumerate(per_axis):
        j = torch.arange(0, dim, 2, dtype=torch.float64)
        base = theta * scaling["factor"] ** (dim / (dim - 2)) if kind == "ntk" else theta
        inv = base ** (-j / dim)
        if kind == "linear":
            inv = inv / scaling["factor"]
        if kind == "llama3":
            turns = scaling["original_max_position_embeddings"] * inv / (2 * math.pi)
            lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
            keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
            inv = keep * inv + (1 - keep) * inv / scaling["factor"]
        if kind == "yarn":
            n = scaling["original_max_position_embeddings"]
            edge = [dim * math.log(n / (beta * 2 * math.pi)) / (2 * math.log(theta)) for beta in (32.0, 1.0)]
            lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), dim - 1)
            ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
            inv = (1 - ramp) * inv + ramp * inv / scaling["factor"]
            amplitude = 0.1 * math.log(scaling["factor"]) + 1
        inverse.append(inv)
        axis += [a] * (dim // 2)
    return (torch.cat(inverse).cuda(), torch.tensor(axis, device="cuda")), amplitude


def _tables(state):
    (inverse, axis), amplitude = state["inverse"], state["amplitude"]
    pos = state["positions"].double()
    if state["case"]["frames"]:
        angle = pos[axis].t()[None] * inverse             # [1, tokens, pairs]
    else:
        angle = pos[..., None] * inverse                  # [batch, tokens, pairs]
    return ((amplitude * angle.cos()).float()[:, None], (amplitude * angle.sin()).float()[:, None])


def _turned(x, cos, sin, case, back=False):
    """Rotates the first ``rotary_dim`` elements of ``x`` (32 bits) by the tables' angles, or back."""
    r = case["rotary_dim"]
    sin = -sin if back else sin
    head, rest = x[..., :r], x[..., r:]
    if case["layout"] == "half":
        a, b = head[..., :r // 2], head[..., r // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)


def _plain_rotary(state):
    case = state["case"]
    cos, sin = _tables(state)
    dt = state["q"].dtype
    out, eps = {}, 1e-6
    for n in ("q", "k"):
        x = state[n].float()
        if case["op"] == "norm_rotary":
            rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
            hat, w = x * rstd, state[n + "_weight"].float()
            out[n] = _turned(hat * w, cos, sin, case).to(dt)
        else:
            out[n] = _turned(x, cos, sin, case).to(dt)
        if case["train"]:
            g = _turned(state["g" + n].float(), cos, sin, case, back=True)
            if case["op"] == "norm_rotary":
                out["d" + n + "_weight"] = (g * hat).sum((0, 1, 2)).to(dt)
                g = g * w
                g = rstd * (g - hat * (g * hat).mean(-1, keepdim=True))
            out["d" + n] = g.to(dt)
    return out


# ------------------------------------------------------------------------------------------------ plain forms: attention

def _seen(case, state, samples, lo, hi):
    """Which keys the queries of ``samples`` see, ``[samples or 1, 1, queries, keys]``; positions ``lo .. hi`` of a packed sequence."""
    n, m = case["queries"], case["keys"]
    i = torch.arange(n, device="cuda")[lo:hi, None] if not case["cache"] else torch.arange(n, device="cuda")[:, None]
    j = torch.arange(m, device="cuda")[None, lo:hi] if not case["cache"] else torch.arange(m, device="cuda")[None]
    if case["cache"]:
        length = state["lengths"][samples].long()[:, None, None]
        return ((j < length) & (j <= length - n + i))[:, None]
    if case["documents"]:
        off = state["offsets"][samples].long()
        doc = torch.searchsorted(off, torch.arange(n, device="cuda").repeat(off.shape[0], 1), right=True) - 1     # behind the last: its number
        start = off.gather(1, doc.clamp_max(off.shape[1] - 1))
        inside = doc < off.shape[1] - 1
        d = doc[:, lo:hi]
        see = (d[:, :, None] == d[:, None, :]) & inside[:, lo:hi, None] & inside[:, None, lo:hi]
        start = start[:, lo:hi, None]
    else:
        see = torch.ones(1, hi - lo, hi - lo, dtype=torch.bool, device="cuda")
        start = 0
    if case["causal"]:
        see = see & ((j <= i) | (j - start < case["prefix"]))
    return see[:, None]


def _distance(case, state, samples, lo, hi):
    i, j = torch.arange(lo, hi, device="cuda")[:, None], torch.arange(lo, hi, device="cuda")[None]
    if case["cache"]:
        i = torch.arange(case["queries"], device="cuda")[:, None] + (state["lengths"][samples].long() - case["queries"])[:, None, None]
        j = torch.arange(case["keys"], device="cuda")[None]
    return (j - i).clamp(-case["distances"], case["distances"]) + case["distances"]


def _sum_by_distance(ds, R):
    """Sums of ``ds [batch, heads, n, n]`` along its diagonals, the far ones joined: ``[heads, 2 R + 1]``."""
    n = ds.shape[-1]
    skew = torch.nn.functional.pad(ds.sum(0).flip(1), (0, n)).flatten(1)[:, :-n].view(ds.shape[1], n, 2 * n - 1).sum(1)
    mid = n - 1                                                   # the column of distance 0
    out = torch.zeros(ds.shape[1], 2 * R + 1, device=ds.device)
    near = min(R, n - 1)
    out[:, R - near:R + near + 1] = skew[:, mid - near:mid + near + 1]
    if n - 1 > R:
        out[:, 0] += skew[:, :mid - R].sum(1)
        out[:, 2 * R] += skew[:, mid + R + 1:].sum(1)
    return out


def _plain_attention(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    B, hq, n, D = q.shape
    hk, m = k.shape[1], k.shape[2]
    G, cap, R = hq // hk, case["softcap"], case["distances"]
    scale = 1.0 / 8 if R else D ** -0.5
    out = torch.zeros(B, n, hq, D, dtype=q.dtype, device="cuda")
    res = {"out": out.view(B, n, hq * D)}
    if case["train"]:
        dq, dk, dv = (torch.zeros(t.shape, dtype=t.dtype, device="cuda") for t in (q, k, v))
        dout = state["gout"].view(B, n, hq, D).transpose(1, 2)
        res.update(dq=dq, dk=dk, dv=dv)
        if R:
            res["dbias"] = torch.zeros(hq, 2 * R + 1, device="cuda")
    # long packed sequences document by document, the rest whole, as many heads at a time as a gigabyte of scores holds
    if case["documents"] and n > 2048:
        parts = [(slice(b, b + 1), lo, hi) for b, off in enumerate(state["cuts"]) for lo, hi in zip(off, off[1:])]
    else:
        parts = [(slice(0, B), 0, max(n, m))]
    for samples, lo, hi in parts:
        nq, nk = min(hi, n) - lo, min(hi, m) - lo
        nb = samples.stop - samples.start
        step = max(1, min(hk, 2 ** 28 // (nb * G * nq * nk)))
        see = _seen(case, state, samples, lo, hi)[:, :, None]             # [samples, 1, 1, queries, keys]
        for h in range(0, hk, step):
            kv, qh = slice(h, h + step), slice(h * G, (h + step) * G)
            hs = min(step, hk - h)
            qf = q[samples, qh, lo:hi].float().reshape(nb, hs, G, nq, D)
            kf, vf = k[samples, kv, lo:hi].float()[:, :, None], v[samples, kv, lo:hi].float()[:, :, None]
            s = (qf @ kf.transpose(-1, -2)) * scale
            if cap:
                t = torch.tanh(s / cap)
                s = cap * t
            if R:
                table = state["bias"].detach()[qh].view(hs, G, -1)
                at = _distance(case, state, samples, lo, hi)
                s = s + (table[:, :, at].permute(2, 0, 1, 3, 4) if at.dim() == 3 else table[:, :, at][None])
            s = s.masked_fill(~see, float("-inf"))
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
            del s
            o = p @ vf
            out[samples, lo:hi, qh] = o.reshape(nb, hs * G, nq, D).transpose(1, 2).to(out.dtype)
            if not case["train"]:
                continue
            do = dout[samples, qh, lo:hi].float().reshape(nb, hs, G, nq, D)
            dv[samples, kv, lo:hi] = (p.transpose(-1, -2) @ do).sum(2).to(dv.dtype)
            ds = p * (do @ vf.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
            del p
            if R:
                res["dbias"][qh] += _sum_by_distance(ds.reshape(nb, hs * G, nq, nk), R)
            if cap:
                ds = ds * (1 - t * t)
                del t
            dq[samples, qh, lo:hi] = (scale * (ds @ kf)).reshape(nb, hs * G, nq, D).to(dq.dtype)
            dk[samples, kv, lo:hi] = (scale * (ds.transpose(-1, -2) @ qf)).sum(2).to(dk.dtype)
    return res


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    st = _inputs(case, seed)
    return _exact_attention(case, st) if case["op"] == "attention" else _exact_rotary(case, st)


def _exact_rotary(case, st):
    """Pair by pair: ``(a, b) -> amplitude * (a cos - b sin, b cos + a sin)`` with the angle of the pair's position and frequency."""
    scaling = _scaling(case) or {"rope_type": "none"}
    kind, f = scaling["rope_type"], scaling.get("factor", 1.0)
    amplitude = 0.1 * math.log(f) + 1 if kind == "yarn" else 1.0
    q, k = st["q"].double(), st["k"].double()
    names = ("q", "k")
    norm = case["op"] == "norm_rotary"
    hats, rstds, outs, grads = {}, {}, {}, {}
    for n, x in zip(names, (q, k)):
        if norm:
            rstds[n] = 1 / torch.sqrt(x.square().mean(-1) + 1e-6)
            hats[n] = x * rstds[n][..., None]
            x = hats[n] * st[n + "_weight"].double()
        outs[n] = x.clone()
        if case["train"]:
            grads[n] = st["g" + n].double().clone()
    first, r = 0, case["rotary_dim"]
    for a, dim in enumerate(_axes(case) or (r,)):
        for j in range(dim // 2):
            if kind == "ntk":
                w = math.exp(-2 * j / dim * (math.log(case["theta"]) + dim / (dim - 2) * math.log(f)))
            else:
                w = math.exp(-2 * j / dim * math.log(case["theta"]))
            if kind == "linear":
                w /= f
            elif kind == "llama3":
                wave, n0 = 2 * math.pi / w, scaling["original_max_position_embeddings"]
                lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
                if wave > n0 / lo:
                    w /= f
                elif wave >= n0 / hi:
                    s = (n0 / wave - lo) / (hi - lo)
                    w = (1 - s) * w / f + s * w
            elif kind == "yarn":
                n0 = scaling["original_max_position_embeddings"]
                def place(turns):
                    return dim * math.log(n0 / (turns * 2 * math.pi)) / (2 * math.log(case["theta"]))
                lo, hi = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), dim - 1)
                s = min(max((j - lo) / max(hi - lo, 0.001), 0.0), 1.0)
                w = w / f * s + w * (1 - s)
            pos = st["positions"].double()
            angle = (pos[a][None] if case["frames"] else pos) * w
            c, s = amplitude * torch.cos(angle)[:, None], amplitude * torch.sin(angle)[:, None]
            pair = first + j
            x0, x1 = (pair, pair + r // 2) if case["layout"] == "half" else (2 * pair, 2 * pair + 1)
            for n in names:
                u, v = outs[n][..., x0].clone(), outs[n][..., x1].clone()
                outs[n][..., x0], outs[n][..., x1] = u * c - v * s, v * c + u * s
                if case["train"]:
                    u, v = grads[n][..., x0].clone(), grads[n][..., x1].clone()
                    grads[n][..., x0], grads[n][..., x1] = u * c + v * s, v * c - u * s
        first += dim // 2
    res = dict(outs)
    if case["train"]:
        for n in names:
            g = grads[n]
            if norm:
                res["d" + n + "_weight"] = torch.einsum("bhsd,bhsd->d", g, hats[n])
                g = g * st[n + "_weight"].double()
                along = torch.einsum("bhsd,bhsd->bhs", g, hats[n]) / case["head_dim"]
                g = rstds[n][..., None] * (g - hats[n] * along[..., None])
            res["d" + n] = g
    return res


def _exact_attention(case, st):
    """Rows of queries in blocks against the keys that they see, head by head."""
    q, k, v = st["q"], st["k"], st["v"]
    B, hq, n, D = q.shape
    hk = k.shape[1]
    G, R, cap = hq // hk, case["distances"], case["softcap"]
    scale = 0.125 if R else 1 / math.sqrt(D)
    first, behind = (t.cuda() for t in _runs(case))
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device="cuda")
    out = torch.zeros(B, n, hq, D, dtype=torch.float64, device="cuda")
    res = {"out": out.view(B, n, hq * D)}
    if case["train"]:
        res.update(dq=zeros(q), dk=zeros(k), dv=zeros(v))
        if R:
            res["dbias"] = torch.zeros(hq, 2 * R + 1, dtype=torch.float64, device="cuda")
    at0 = [x - n for x in _cache_lengths(case)] if case["cache"] else [0] * B
    block = 4096
    for b in range(B):
        for r0 in range(0, n, block):
            r1 = min(n, r0 + block)
            lo, hi = first[b, r0:r1], behind[b, r0:r1]
            some = hi > lo
            if not bool(some.any()):
                continue
            k0, k1 = int(lo[some].min()), int(hi.max())
            j = torch.arange(k0, k1, device="cuda")
            hidden = (j[None] < lo[:, None]) | (j[None] >= hi[:, None])
            far = j[None] - (torch.arange(r0, r1, device="cuda") + at0[b])[:, None]
            for h in range(hq):
                Q, K, V = q[b, h, r0:r1].double(), k[b, h // G, k0:k1].double(), v[b, h // G, k0:k1].double()
                raw = (Q @ K.T) * scale
                s = cap * torch.tanh(raw / cap) if cap else raw
                if R:
                    s = s + st["bias"][h].double()[far.clamp(-R, R) + R]
                s = torch.where(hidden, -math.inf, s)
                p = torch.softmax(s, -1)
                p = torch.where(some[:, None], p, torch.zeros_like(p))
                o = p @ V
                out[b, r0:r1, h] = o
                if not case["train"]:
                    continue
                do = st["gout"].view(B, n, hq, D)[b, r0:r1, h].double()
                res["dv"][b, h // G, k0:k1] += p.T @ do
                dp = do @ V.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                if R:
                    res["dbias"][h] += torch.bincount((far.clamp(-R, R) + R).flatten(), weights=ds.flatten(), minlength=2 * R + 1)
                if cap:
                    ds = ds * (1 - torch.tanh(raw / cap) ** 2)
                res["dq"][b, h, r0:r1] = scale * (ds @ K)
                res["dk"][b, h // G, k0:k1] += scale * (ds.T @ Q)
    return res
