"""``ops.masked_attention`` on the GPU against 64 bits: masks, heads, strides, caps, biases, gradients."""

import pytest
import torch

from attention_oracle import attention, close, runs
from teletron_b200 import ops
from teletron_b200.ops import _lib, status

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def heads(B, S, counts, D, dtype, token_major):
    if token_major:
        buf = torch.randn(B, S, sum(counts) * D, device="cuda").to(dtype)
        return [p.view(B, S, c, D).transpose(1, 2) for p, c in zip(buf.split([c * D for c in counts], dim=-1), counts)]
    return [torch.randn(B, c, S, D, device="cuda").to(dtype) for c in counts]


def operands(B, n, m, hq, hk, D, dtype, token_major=True):
    if n == m:
        return heads(B, n, (hq, hk, hk), D, dtype, token_major)
    return heads(B, n, (hq,), D, dtype, token_major) + heads(B, m, (hk, hk), D, dtype, token_major)


def check(B, n, m, hq, hk, D, dtype, token_major=True, train=True, scale=None, softcap=None, R=None, spoil=True, tensors=None, **mask):
    torch.manual_seed(0)
    q, k, v = tensors or operands(B, n, m, hq, hk, D, dtype, token_major)
    ranges = ops.key_ranges(n, m, batch=B, device="cuda", **mask)
    bias = None if R is None else (0.7 * torch.randn(hq, 2 * R + 1, device="cuda")).requires_grad_(train)
    first, behind = ranges.first.long(), ranges.behind.long()
    start = ranges.query_start
    dout = torch.randn(B, n, hq * D, device="cuda").to(dtype)
    if spoil:       # whatever no run reaches holds NaN and infinities
        j = torch.arange(m, device="cuda")
        used = ((j >= first[..., None]) & (j < behind[..., None])).any(1)
        live = first < behind
        for t, keep in ((q, live), (k, used), (v, used)):
            t.masked_fill_(~keep[:, None, :, None], float("nan"))
        dout.masked_fill_(~live[..., None], float("inf"))
    leaves = [t.requires_grad_(train) for t in (q, k, v)] + ([bias] if R is not None else [])
    out = ops.masked_attention(q, k, v, ranges, scale=scale, softcap=softcap, distance_bias=bias)
    assert out.shape == (B, n, hq * D) and out.dtype == dtype and out.is_contiguous()
    grads = torch.autograd.grad(out, leaves, dout) if train else ()
    status.check_all(what="test")
    by_head = lambda t: t.view(B, n, hq, D).transpose(1, 2)
    want = attention(*[t.detach() for t in (q, k, v)], first, behind, D ** -0.5 if scale is None else scale, dtype, softcap,
                     None if bias is None else bias.detach(), start, by_head(dout) if train else None)
    close(by_head(out.detach()), want["out"], "out")
    for name, g in zip(("dq", "dk", "dv", "dbias"), grads):
        close(g, want[name], name)
    return out


MASKS = {
    "all": {}, "causal": dict(causal=True), "prefix": dict(causal=True, prefix_len=37), "length": dict(kv_valid_len=150), "nothing": dict(kv_valid_len=0),
    "documents": dict(documents=[3, 40, 40, 129, 200, 290]), "causal documents": dict(causal=True, documents=[0, 128, 256, 299], prefix_len=70),
    "one document": dict(documents=[0, 131]), "tail document": dict(documents=[270, 300])}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mask", list(MASKS))
def test_masks(mask, D):
    check(2, 300, 300, 4, 2, D, BF16, **MASKS[mask])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (6, 2), (4, 1), (8, 2)])
@pytest.mark.parametrize("token_major", [True, False])
def test_heads_types_and_layouts(hq, hk, dtype, token_major):
    check(2, 150, 150, hq, hk, 64, dtype, token_major, causal=True)
    check(1, 140, 140, hq, hk, 128, dtype, token_major, documents=[0, 130])


@pytest.mark.parametrize("n,m", [(1, 1), (1, 128), (1, 129), (2, 1000), (127, 127), (128, 128), (129, 129), (255, 513), (256, 256), (257, 385), (640, 640)])
def test_lengths(n, m):
    check(1, n, m, 2, 1, 128, BF16)
    check(1, n, m, 2, 2, 64, FP16)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16)])
def test_caches(D, dtype):
    check(4, 1, 700, 8, 2, D, dtype, causal=True, kv_valid_len=torch.tensor([700, 1, 129, 400], device="cuda"),
          query_start=torch.tensor([699, 0, 128, 399], device="cuda"))
    check(3, 5, 300, 4, 4, D, dtype, causal=True, kv_valid_len=torch.tensor([300, 5, 3], device="cuda"), query_start=torch.tensor([295, 0, -2], device="cuda"), R=40)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("scale", [None, 0.5, 0.0, -0.1])
@pytest.mark.parametrize("softcap", [None, 3.0, 50.0])
def test_scales_and_caps(D, dtype, scale, softcap):
    check(1, 200, 200, 4, 2, D, dtype, scale=scale, softcap=softcap, causal=True, prefix_len=20)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16)])
@pytest.mark.parametrize("R", [0, 1, 40, 128, 300, 1024])
def test_distance_bias(D, dtype, R):
    check(2, 300, 300, 4, 4, D, dtype, scale=0.125, R=R, documents=[[0, 300], [0, 211]])
    check(1, 430, 430, 4, 2, D, dtype, R=R, causal=True, softcap=20.0)


def test_bias_of_many_tiles():
    check(1, 1300, 1300, 2, 2, 64, BF16, R=128, scale=0.125)
    check(1, 1300, 1300, 2, 2, 64, BF16, R=700, scale=0.125, train=False)


def test_several_seeds_of_ragged_masks():
    g = torch.Generator().manual_seed(5)
    for _ in range(6):
        n = int(torch.randint(1, 700, (1,), generator=g))
        cuts = torch.randint(0, n + 1, (3, 5), generator=g).sort(1).values
        check(3, n, n, 4, 2, 128, BF16, documents=cuts, causal=bool(torch.randint(0, 2, (1,), generator=g)))


def test_runs_on_the_device_are_the_definitions():
    from test_masked_attention_cpu import CASES, expected
    for kw in CASES:
        got = ops.key_ranges(**kw, device="cuda")
        first, behind = expected(kw)
        assert torch.equal(got.first.cpu(), first) and torch.equal(got.behind.cpu(), behind), kw
        assert got.plan is not None


def test_lengths_beyond_32_bits_and_batches_beyond_a_grid():
    huge = 2 ** 32 + 1
    for kw in (dict(prefix_len=huge), dict(query_start=huge), dict(query_start=-huge), dict(kv_valid_len=torch.tensor([huge, 3])),
               dict(documents=[2, huge]), dict(prefix_len=[huge, 1])):
        for a, b in zip(*[(r.first.cpu(), r.behind.cpu()) for r in (ops.key_ranges(150, batch=2, causal=True, device=d, **kw) for d in ("cuda", "cpu"))]):
            assert torch.equal(a, b), kw
    from teletron_b200.ops import fallback
    q = torch.randn(65537, 1, 2, 64, device="cuda").to(BF16)
    was = fallback.strict()
    try:
        fallback.set_strict(False)
        got = ops.masked_attention(q, q, q, ops.key_ranges(2, batch=65537, causal=True, device="cuda"))
    finally:
        fallback.set_strict(was)
    assert torch.equal(got[:, 0], q[:, 0, 0])


def test_large_scores_and_infinite_biases():
    torch.manual_seed(1)
    q, k, v = heads(1, 200, (2, 2, 2), 64, BF16, False)
    # scores up to about 60: weights of 1 and 0, and maxima that grow from tile to tile
    check(1, 200, 200, 2, 2, 64, BF16, scale=2.0, tensors=(q, k, v))
    bias = torch.zeros(2, 2 * 70 + 1, device="cuda")
    bias[:, 0] = bias[:, -1] = float("-inf")                # a window of 69 on both sides
    out = ops.masked_attention(q.detach(), k.detach(), v.detach(), ops.key_ranges(200, device="cuda"), distance_bias=bias)
    i = torch.arange(200, device="cuda")
    first, behind = (i - 69).clamp_min(0)[None], (i + 70).clamp_max(200)[None]
    close(out.view(1, 200, 2, 64).transpose(1, 2), attention(q.detach(), k.detach(), v.detach(), first, behind, 0.125, BF16)["out"])
    bias[:] = float("-inf")
    assert not bool(ops.masked_attention(q.detach(), k.detach(), v.detach(), ops.key_ranges(200, device="cuda"), distance_bias=bias).any())


@pytest.mark.parametrize("softcap", [1e-2, 1e-6, 1e-9])
def test_caps_far_below_the_scores(softcap):
    """All weights of a row nearly or wholly the same: behind the cap no score is more than it from another."""
    torch.manual_seed(7)
    q, k, v = heads(1, 140, (2, 1, 1), 64, BF16, False)
    q[:, :, 3] = 0
    out = ops.masked_attention(q, k, v, ops.key_ranges(140, causal=True, device="cuda"), softcap=softcap)
    mean = v.double().cumsum(2) / torch.arange(1, 141, device="cuda")[:, None]
    got = out.view(1, 140, 2, 64).transpose(1, 2).double()
    size = v.double().abs().cumsum(2) / torch.arange(1, 141, device="cuda")[:, None]
    # weights off by e^(2 cap), P and the output rounded to 2^-8 each
    assert bool(((got - mean).abs() <= (2.5 * softcap + 2 * 2.0 ** -8) * size + 2.0 ** -8 * mean.abs()).all())


def test_strides_that_copies_cannot_address():
    torch.manual_seed(2)
    base = torch.randn(1, 2, 130, 65, device="cuda").to(BF16)
    q = base[..., 1:]                                       # rows at odd addresses
    k = torch.randn(1, 1, 130, 64, device="cuda").to(BF16).expand(1, 2, 130, 64)       # one row of heads for both
    v = torch.randn(1, 2, 64, 130, device="cuda").to(BF16).transpose(2, 3)
    r = ops.key_ranges(130, causal=True, device="cuda")
    want = ops.masked_attention(q.contiguous(), k.contiguous(), v.contiguous(), r)
    assert torch.equal(ops.masked_attention(q, k, v, r), want)
    far = torch.randn(1, 2, 4096, 64, device="cuda").to(BF16)[:, :, ::32][:, :, :128]          # every 32nd row
    r = ops.key_ranges(128, device="cuda")
    assert torch.equal(ops.masked_attention(far, far, far, r), ops.masked_attention(*[far.contiguous()] * 3, r))


def test_results_do_not_depend_on_the_run():
    torch.manual_seed(3)
    q, k, v = (t.requires_grad_() for t in heads(2, 520, (4, 2, 2), 128, BF16, True))
    bias = torch.randn(4, 129, device="cuda", requires_grad=True)
    r = ops.key_ranges(520, batch=2, causal=True, device="cuda")
    dout = torch.randn(2, 520, 512, device="cuda").to(BF16)

    def step():
        out = ops.masked_attention(q, k, v, r, distance_bias=bias)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v, bias), dout))

    a, b = step(), step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_difference_of_the_forward_is_the_gradient():
    """Along a direction in which the output moves by far more than it is rounded."""
    torch.manual_seed(4)
    q, k, v = (t.float() for t in heads(1, 160, (2, 1, 1), 64, BF16, False))
    r = ops.key_ranges(160, causal=True, device="cuda")
    dout = torch.randn(1, 160, 128, device="cuda").to(BF16)
    leaves = [t.to(BF16).requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.masked_attention(*leaves, r, softcap=5.0), leaves, dout)
    for i in range(3):
        d = grads[i].float() / grads[i].float().norm()          # along the gradient itself
        ends, moved_by = [], []
        for s in (1.0, -1.0):
            moved = [t.detach() for t in leaves]
            moved[i] = (leaves[i].detach().float() + s * d).to(BF16)
            moved_by.append(moved[i].float() - leaves[i].detach().float())
            ends.append((ops.masked_attention(*moved, r, softcap=5.0).double() * dout.double()).sum())
        along = float((grads[i].double() * (moved_by[0] - moved_by[1]).double()).sum())
        # outputs rounded to 2^-8: 20480 of them, sizes near 1, against dout near 1: a deviation of about sqrt(20480) 2^-8 / 1.7 = 0.33
        # on either side; five of those
        assert abs(float(ends[0] - ends[1]) - along) <= 5 * 0.33 * 2 ** 0.5 + 0.05 * abs(along), i


def test_streams_and_captured_graphs():
    torch.manual_seed(5)
    q, k, v = heads(2, 300, (4, 2, 2), 64, BF16, True)
    bias = torch.randn(4, 65, device="cuda")
    offsets = torch.tensor([[0, 300], [0, 210]], device="cuda", dtype=torch.int32)
    dout = torch.randn(2, 300, 256, device="cuda").to(BF16)

    def step():
        r = ops.key_ranges(300, batch=2, documents=offsets, causal=True)
        leaves = [t.detach().requires_grad_() for t in (q, k, v, bias)]
        out = ops.masked_attention(*leaves[:3], r, distance_bias=leaves[3])
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graphs, held = [], []
    for _ in range(2):              # two graphs of their own, replayed one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step())
        graphs.append(g)
    q.copy_(torch.randn_like(q))
    offsets[1, 1] = 77
    for g in graphs:
        g.replay()
    again = step()
    for h in held:
        assert all(torch.equal(a, b) for a, b in zip(h, again))
    assert not torch.equal(held[0][0], want[0]) and not bool(held[0][0][1, 77:].any())


def test_what_the_kernels_do_not_take_runs_plain_with_a_note():
    from teletron_b200.ops import fallback
    q = torch.randn(1, 2, 9, 80, device="cuda", dtype=BF16)
    r = ops.key_ranges(9, device="cuda")
    was = fallback.strict()
    try:
        fallback.set_strict(False)
        n = sum(fallback.SEEN.values())
        assert ops.masked_attention(q, q, q, r).shape == (1, 9, 160) and sum(fallback.SEEN.values()) == n + 1
        fallback.set_strict(True)
        with pytest.raises(fallback.LibraryFallbackError):
            ops.masked_attention(q, q, q, r)
    finally:
        fallback.set_strict(was)
    x = torch.randn(1, 2, 9, 64, device="cuda")             # fp32: the plain path, as for the other ops
    assert ops.masked_attention(x, x, x, r).dtype == torch.float32
    before = _lib.LAUNCHES
    h = x.to(FP16)
    ops.masked_attention(h, h, h, r)
    assert _lib.LAUNCHES == before + 1
    with pytest.raises(ValueError):
        ops.masked_attention(h, h, h, ops.key_ranges(9))    # runs on the CPU


def test_projection_rotation_and_attention_together():
    """A layer as it is used: a fused projection's views, rotated, attended to and differentiated, against 64 bits of the same layer."""
    torch.manual_seed(6)
    B, n, hq, hk, D, C = 2, 200, 4, 2, 64, 256
    x = torch.randn(B, n, C, device="cuda").to(BF16).requires_grad_()
    w = (torch.randn((hq + 2 * hk) * D, C, device="cuda") / 16).to(BF16).requires_grad_()
    lengths = torch.tensor([[0, 200], [0, 150]], device="cuda")
    freqs = ops.rotary_frequencies(D, 500000.0, device="cuda")
    pos = torch.arange(n, device="cuda")
    dout = torch.randn(B, n, hq * D, device="cuda").to(BF16)
    qkv = ops.linear(x, w)
    q, k, v = (t.view(B, n, -1, D).transpose(1, 2) for t in qkv.split([hq * D, hk * D, hk * D], dim=-1))
    q, k = ops.rotary(q, k, pos, freqs)
    out = ops.masked_attention(q, k, v, ops.key_ranges(n, batch=B, causal=True, documents=lengths), softcap=30.0)
    got = (out, *torch.autograd.grad(out, (x, w), dout))
    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    q, k, v = (t.view(B, n, -1, D).transpose(1, 2) for t in (xd @ wd.T).split([hq * D, hk * D, hk * D], dim=-1))
    with ops.impl("torch"):
        q, k = ops.rotary(q, k, pos, freqs)
        ref = ops.masked_attention(q, k, v, ops.key_ranges(n, batch=B, causal=True, documents=lengths), softcap=30.0)
    want = (ref, *torch.autograd.grad(ref, (xd, wd), dout.double()))
    for a, b in zip(got, want):
        # nine roundings to 2^-8 between input and gradient, each of independent elements: a relative norm of 9 * 2^-8 bounds them all
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 9 * 2 ** -8


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, FP16), (128, BF16)])
@pytest.mark.parametrize("n,hq,hk", [(1, 1, 1), (1, 32, 1), (2, 32, 2), (16, 2, 2), (17, 1, 1), (32, 2, 2), (33, 2, 2), (5, 24, 4)])
def test_few_queries(n, hq, hk, D, dtype):
    """Both sides of the borders between the kernels for few queries (16 and 32 rows of a group) and the one for tiles."""
    lengths = torch.tensor([1500, n, 700], device="cuda")
    kw = dict(causal=True, kv_valid_len=lengths, query_start=lengths - n)
    check(3, n, 1500, hq, hk, D, dtype, train=False, **kw)
    check(3, n, 1500, hq, hk, D, dtype, R=60, softcap=8.0, scale=-0.2, **kw)
    check(2, n, n, hq, hk, D, dtype, documents=[0, (n + 1) // 2, n], causal=True)
    check(2, n, 300, hq, hk, D, dtype, False, kv_valid_len=torch.tensor([0, 299], device="cuda"))


def test_few_queries_over_one_long_cache():
    check(1, 1, 40000, 4, 1, 64, BF16, train=False, causal=True, query_start=39999)
    check(1, 3, 20001, 2, 2, 128, BF16, train=False, causal=True, query_start=20000 - 2, token_major=False)


def test_few_queries_past_32_bits_of_elements():
    """A cache whose last rows lie beyond 2^32 elements: two samples, far apart in one allocation."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("not enough device memory")
    far = 2 ** 32 // (2 * 64) + 8
    buf = torch.empty(far * 2 * 64 + 600 * 2 * 64, device="cuda", dtype=BF16)
    k = torch.as_strided(buf, (2, 2, 300, 64), (far * 2 * 64, 64, 128, 1))
    k.copy_(torch.randn(2, 2, 300, 64, device="cuda"))
    q = torch.randn(2, 4, 1, 64, device="cuda").to(BF16)
    r = ops.key_ranges(1, 300, batch=2, causal=True, query_start=299, device="cuda")
    assert torch.equal(ops.masked_attention(q, k, k, r), ops.masked_attention(q, k.contiguous(), k.contiguous(), r))
    q = torch.randn(2, 4, 300, 64, device="cuda").to(BF16)
    r = ops.key_ranges(300, batch=2, causal=True, device="cuda")
    assert torch.equal(ops.masked_attention(q, k, k, r), ops.masked_attention(q, k.contiguous(), k.contiguous(), r))


def test_new_tokens_in_a_captured_graph_and_on_two_streams():
    torch.manual_seed(11)
    B, hq, hk, n, D = 3, 8, 2, 5000, 128
    q = torch.randn(B, hq, 1, D, device="cuda").to(BF16)
    k, v = (torch.randn(B, hk, n, D, device="cuda").to(BF16) for _ in range(2))
    lengths = torch.tensor([5000, 40, 1300], device="cuda")

    def step(x):            # a layer after the other: each reads what the one ahead wrote
        r = ops.key_ranges(1, n, batch=B, causal=True, kv_valid_len=lengths, query_start=lengths - 1)
        for _ in range(4):
            x = ops.masked_attention(x, k, v, r, scale=1.0).view(B, 1, hq, D).transpose(1, 2)
        return x

    want = step(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(q)
    for _ in range(3):
        graph.replay()
    assert torch.equal(held, want)
    lengths.copy_(torch.tensor([0, 5000, 4999], device="cuda"))
    q.neg_()
    for _ in range(3):
        graph.replay()
    want = step(q)
    assert torch.equal(held, want) and not bool(want[0].any())
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step(q))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("batch", [128, 129])
def test_few_queries_of_many_samples(batch):
    """Both sides of the largest batch whose steps are dealt out."""
    lengths = torch.arange(batch, device="cuda") * 5
    check(batch, 1, 600, 2, 1, 64, BF16, train=False, causal=True, kv_valid_len=lengths, query_start=lengths - 1)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("batch,hk,group,n,m", [(1, 2, 8, 4, 1700), (2, 3, 20, 1, 2500), (40, 8, 4, 1, 2500), (70, 8, 2, 9, 300), (37, 8, 32, 1, 700),
                                                (1, 1, 17, 1, 1536), (1, 1, 17, 1, 1537), (75, 1, 32, 1, 600)])
def test_few_queries_by_shares_and_by_heads(batch, hk, group, n, m, D):
    """Few and many samples and key heads, on either side of what makes shares of them, with one and with two tiles of rows."""
    torch.manual_seed(batch + m)
    lengths = torch.randint(n, m + 1, (batch,), device="cuda")
    lengths[0] = m
    check(batch, n, m, hk * group, hk, D, BF16, train=False, causal=True, kv_valid_len=lengths, query_start=lengths - n)


def test_broadcast_inputs_and_inputs_given_twice():
    torch.manual_seed(12)
    freqs, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(150, device="cuda")
    r = ops.key_ranges(150, batch=2, causal=True, device="cuda")
    x = torch.randn(2, 2, 150, 64, device="cuda").to(BF16).requires_grad_()
    one = torch.randn(1, 1, 150, 64, device="cuda").to(BF16).requires_grad_()
    dout = torch.randn(2, 150, 128, device="cuda").to(BF16)

    def run(q, k, v):
        q, k = ops.rotary(q, k, pos, freqs)
        return ops.masked_attention(q, k, v, r)

    shared = run(x, one.expand(2, 2, -1, -1), one.expand(2, 1, -1, -1).expand(2, 2, -1, -1))
    got = torch.autograd.grad(shared, (x, one), dout)
    k, v = (one.detach().repeat(2, 2, 1, 1).requires_grad_() for _ in range(2))
    own = run(x, k, v)
    dx, dk, dv = torch.autograd.grad(own, (x, k, v), dout)
    assert torch.equal(shared, own) and torch.equal(got[0], dx)
    # autograd adds the four copies' gradients, and those of both operands, in bf16
    want, size = (f(dk.double()) + f(dv.double()) for f in (lambda t: t.sum((0, 1), keepdim=True), lambda t: t.abs().sum((0, 1), keepdim=True)))
    assert bool(((got[1].double() - want).abs() <= 6 * 2.0 ** -8 * size).all())
    same, = torch.autograd.grad(run(x, x, x), x, dout)
    q, k, v = (x.detach().clone().requires_grad_() for _ in range(3))
    parts = [g.double() for g in torch.autograd.grad(run(q, k, v), (q, k, v), dout)]
    assert bool(((same.double() - sum(parts)).abs() <= 2 * 2.0 ** -8 * sum(g.abs() for g in parts)).all())


def test_a_captured_backward_while_an_eager_graph_of_the_same_leaves_lives():
    torch.manual_seed(13)
    freqs, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(150, device="cuda")
    r = ops.key_ranges(150, causal=True, device="cuda")
    leaves = [torch.randn(1, 2, 150, 64, device="cuda").to(BF16).requires_grad_() for _ in range(3)]
    leaves += [torch.randn(64, device="cuda").to(BF16).requires_grad_() for _ in range(2)] + [torch.randn(2, 41, device="cuda").requires_grad_()]
    dout = torch.randn(1, 150, 128, device="cuda").to(BF16)

    def forward():
        q, k = ops.qk_norm_rotary(*leaves[:2], *leaves[3:5], pos, freqs)
        return ops.masked_attention(q, k, leaves[2], r, distance_bias=leaves[5])

    # on the stream that is captured: the eager graph's accumulation nodes belong to the stream that they were made on, and the engine
    # makes that one wait for what is captured, whatever the operator is
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(forward(), leaves, dout)
        alive = forward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = torch.autograd.grad(forward(), leaves, dout)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, want))
    with torch.cuda.stream(side):
        again = torch.autograd.grad(alive, leaves, dout)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_a_first_call_in_a_captured_graph(monkeypatch):
    from teletron_b200.ops import gemm_tcgen05
    monkeypatch.setattr(gemm_tcgen05, "_STATUS", {})
    q = torch.randn(1, 2, 150, 64, device="cuda").to(BF16)
    r = ops.key_ranges(150, causal=True, device="cuda")
    word, = gemm_tcgen05._STATUS.values()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.masked_attention(q, q, q, r)
    assert list(gemm_tcgen05._STATUS.values())[0] is word and not bool(word.any())
    graph.replay()
    assert torch.equal(held, ops.masked_attention(q, q, q, r))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,mask", [(1, {}), (129, dict(documents=[0, 128, 129])), (300, dict(documents=list(range(301)))), (130, dict(causal=True, documents=[0, 1, 2, 130])),
                                    (257, dict(causal=True, kv_valid_len=1))])
def test_queries_that_see_one_key_have_no_gradient_of_their_scores(n, mask, D):
    torch.manual_seed(14)
    r = ops.key_ranges(n, batch=2, device="cuda", **mask)
    for softcap, R in ((None, None), (3.0, None), (None, 9)):
        q, k, v = (t.requires_grad_() for t in heads(2, n, (4, 2, 2), D, BF16, True))
        bias = None if R is None else torch.randn(4, 2 * R + 1, device="cuda").requires_grad_()
        out = ops.masked_attention(q, k, v, r, softcap=softcap, distance_bias=bias)
        dout = torch.randn_like(out)
        one = r.behind - r.first == 1
        grads = torch.autograd.grad(out, (q, k, v) + (() if bias is None else (bias,)), dout)
        assert not bool(grads[0].transpose(1, 2)[one].any()) and bool(grads[2].any())
        if bool((one | (r.behind == r.first)).all()):
            assert not bool(grads[1].any()) and (bias is None or not bool(grads[3].any()))


@pytest.mark.parametrize("n", [2, 3, 16, 128, 129])
def test_gradients_of_few_keys(n):
    """dP - delta of few keys is small against both: the gradients are no further off than their own rounding and that of dS."""
    torch.manual_seed(15)
    q, k, v = (t.requires_grad_() for t in heads(4, n, (8, 8, 8), 128, BF16, True))
    r = ops.key_ranges(n, batch=4, causal=True, device="cuda")
    out = ops.masked_attention(q, k, v, r)
    dout = torch.randn_like(out)
    got = torch.autograd.grad(out, (q, k, v), dout)
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]
    with ops.impl("torch"):
        want = torch.autograd.grad(ops.masked_attention(*x, r), x, dout.double())
    for a, b in zip(got, want):
        # two roundings, each off by at most 2^-8 and uniformly spread below that (by 3^-1/2 of it), and for 129 keys delta's
        assert float((a.double() - b).norm() / b.norm()) < (2 if n <= 128 else 3) ** 0.5 * 2.0 ** -8 / 3 ** 0.5


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    freqs, pos, w = ops.rotary_frequencies(64, device="cuda"), torch.arange(9, device="cuda"), torch.ones(64, device="cuda", dtype=BF16)
    q = torch.randn(1, 2, 9, 64, device="cuda").to(BF16)
    runs_ = ops.key_ranges(9, causal=True, device="cuda")
    want = ops.masked_attention(q, q, q, runs_), ops.rotary(q, q, pos, freqs)[0], ops.qk_norm_rotary(q, q, w, w, pos, freqs)[0]
    with fwd.dual_level():
        x = fwd.make_dual(q, torch.ones_like(q))
        for f in (lambda: ops.masked_attention(q, x, q, runs_), lambda: ops.rotary(q, x, pos, freqs), lambda: ops.qk_norm_rotary(x, q, w, w, pos, freqs)):
            with pytest.raises(RuntimeError):
                f()
        got = ops.masked_attention(q, q, q, runs_), ops.rotary(q, q, pos, freqs)[0], ops.qk_norm_rotary(q, q, w, w, pos, freqs)[0]
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    # few rows by themselves and in a tile: P is rounded to bf16 against another maximum, and the output once, in each
    assert torch.allclose(got[0].float(), want[0].float(), atol=4 * 2.0 ** -8 * float(q.float().abs().max()), rtol=0)


@pytest.mark.parametrize("B,n,m", [(0, 3, 3), (2, 0, 3), (2, 3, 0)])
def test_empty_operands_are_no_fallback(B, n, m):
    """No samples, no queries, a cache that holds nothing yet: what a training run with its strict kernels calls too."""
    from teletron_b200.ops import fallback
    q, k, v = (torch.randn(B, h, s, 64, device="cuda").to(BF16).requires_grad_() for h, s in ((4, n), (2, m), (2, m)))
    was = fallback.strict()
    try:
        fallback.set_strict(True)
        out = ops.masked_attention(q, k, v, ops.key_ranges(n, m, batch=B, device="cuda"))
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
    finally:
        fallback.set_strict(was)
    assert out.shape == (B, n, 256) and not bool(out.any()) and all(not bool(g.any()) for g in grads)


def test_two_threads_at_once():
    """Rotation and attention, forward and backward, by two threads on streams of their own: the bits of one alone."""
    import threading
    freqs = ops.rotary_frequencies(64, device="cuda")

    def work(seed, n, hk):
        g = torch.Generator(device="cuda").manual_seed(seed)
        q, k, v = (torch.randn(2, h, n, 64, device="cuda", generator=g).to(BF16).requires_grad_() for h in (4, hk, hk))
        dout = torch.randn(2, n, 256, device="cuda", generator=g).to(BF16)
        new = torch.randn(2, 4, 1, 64, device="cuda", generator=g).to(BF16)
        out = []
        for _ in range(20):
            a, b = ops.rotary(q, k, torch.arange(n, device="cuda"), freqs)
            y = ops.masked_attention(a, b, v, ops.key_ranges(n, batch=2, causal=True, documents=[0, n // 3, n], device="cuda"))
            one = ops.masked_attention(new, b.detach(), v.detach(), ops.key_ranges(1, n, batch=2, device="cuda"))
            out = [y.detach(), one, *torch.autograd.grad(y, (q, k, v), dout)]
        return out

    jobs = [(1, 300, 2), (2, 513, 4)]
    want = [work(*job) for job in jobs]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = work(*jobs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    status.check_all(what="test")
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))
