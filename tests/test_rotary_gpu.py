"""``ops.rotary`` and ``ops.qk_norm_rotary`` on the GPU against 64 bits, forward and backward."""

import pytest
import torch

from rotary_oracle import ROTATION, U32, angles, close, rounding, inverse_frequencies, norm_error, pair_size, turn
from teletron_b200 import ops
from teletron_b200.ops import _lib

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def heads(B, S, counts, D, dtype, layout):
    """Views of one token-major buffer, tensors of their own, or views that start one element behind an aligned address."""
    if layout == "packed":
        buf = torch.randn(B, S, sum(counts) * D, device="cuda").to(dtype)
        return [p.view(B, S, c, D).transpose(1, 2) for p, c in zip(buf.split([c * D for c in counts], dim=-1), counts)]
    if layout == "odd":
        return [torch.randn(B * c * S * D + 1, device="cuda").to(dtype)[1:].view(B, c, S, D) for c in counts]
    return [torch.randn(B, c, S, D, device="cuda").to(dtype) for c in counts]


# (batch, tokens, query heads, key heads, head dim, rotated): every vector width, lane count and ragged share
SHAPES = [(1, 1, 1, 1, 128, 128), (3, 7, 8, 2, 128, 128), (2, 33, 5, 1, 64, 32), (1, 130, 3, 3, 80, 20), (2, 5, 4, 2, 96, 96),
          (1, 9, 2, 1, 256, 64), (1, 6, 3, 1, 40, 10), (1, 3, 2, 2, 8, 2), (1, 4, 40, 8, 128, 64), (1, 5, 1, 1, 254, 250), (2, 700, 12, 4, 64, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["packed", "own", "odd"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(shape, layout, interleaved, dtype):
    B, S, hq, hk, D, rot = shape
    torch.manual_seed(0)
    q, k = heads(B, S, (hq, hk), D, dtype, layout)
    pos = torch.randint(0, 100000, (B, S), device="cuda", dtype=torch.int32)
    freqs = ops.rotary_frequencies(rot, 10000.0, interleaved=interleaved, device="cuda")
    a = angles(pos[:, None], inverse_frequencies(rot, 10000.0))
    q.requires_grad_(), k.requires_grad_()
    before = _lib.LAUNCHES
    outs = ops.rotary(q, k, pos, freqs)
    assert _lib.LAUNCHES == before + 1
    grads = [torch.randn(o.shape, device="cuda").to(dtype) for o in outs]
    dx = torch.autograd.grad(outs, (q, k), grads)
    for x, y, g, d in zip((q, k), outs, grads, dx):
        assert y.is_contiguous() and y.dtype == dtype
        want = turn(x.detach().double(), a, 1.0, interleaved)
        close(y.detach(), want, rounding(dtype, want) + ROTATION * pair_size(x.detach().double(), rot // 2, 1.0, interleaved), "y")
        assert torch.equal(y.detach()[..., rot:], x.detach()[..., rot:])
        want = turn(g.double(), -a, 1.0, interleaved)
        close(d, want, rounding(dtype, want) + ROTATION * pair_size(g.double(), rot // 2, 1.0, interleaved), "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["packed", "odd"])
@pytest.mark.parametrize("shape", SHAPES)
def test_qk_norm_rotary(shape, layout, interleaved, dtype):
    B, S, hq, hk, D, rot = shape
    torch.manual_seed(1)
    q, k = heads(B, S, (hq, hk), D, dtype, layout)
    w = [(1 + 0.2 * torch.randn(D, device="cuda")).to(dtype).requires_grad_() for _ in range(2)]
    pos = torch.randint(0, 100000, (S,), device="cuda")
    freqs = ops.rotary_frequencies(rot, 500000.0, interleaved=interleaved, device="cuda")
    a = angles(pos[None, None], inverse_frequencies(rot, 500000.0))
    q.requires_grad_(), k.requires_grad_()
    outs = ops.qk_norm_rotary(q, k, *w, pos, freqs)
    grads = [torch.randn(o.shape, device="cuda").to(dtype) for o in outs]
    got = torch.autograd.grad(outs, (q, k, *w), grads)
    rel = norm_error(D)
    for i, (x, y, g) in enumerate(zip((q, k), outs, grads)):
        xd, wd, gd = x.detach().double(), w[i].detach().double(), g.double()
        r = torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-6)
        hat = xd * r
        want = turn(hat * wd, a, 1.0, interleaved)
        size = pair_size(hat * wd, rot // 2, 1.0, interleaved)
        close(y.detach(), want, rounding(dtype, want) + (ROTATION + rel) * size, "y")
        back = turn(gd, -a, 1.0, interleaved)
        back_size = pair_size(gd, rot // 2, 1.0, interleaved)
        dw = (back * hat).sum((0, 1, 2))
        rows = x[..., 0].numel()
        # a sum of `rows` products in any order, each with the errors of its factors
        bound = (back_size * hat.abs()).sum((0, 1, 2)) * (rows * U32 + ROTATION + rel)
        close(got[2 + i], dw, rounding(dtype, dw) + bound, "dw")
        gw = back * wd
        dot = (gw * hat).mean(-1, keepdim=True)
        dx = r * (gw - hat * dot)
        spread = r * (back_size * wd.abs() + hat.abs() * (back_size * wd.abs() * hat.abs()).mean(-1, keepdim=True))
        close(got[i], dx, rounding(dtype, dx) + spread * (ROTATION + 3 * rel + D * U32), "dx")


def test_axes_amplitude_and_shared_positions():
    torch.manual_seed(2)
    grid = torch.stack([t.reshape(-1) for t in torch.meshgrid(torch.arange(3), torch.arange(5), torch.arange(7), indexing="ij")]).cuda()
    S = grid.shape[1]
    q, k = torch.randn(2, 3, S, 128, device="cuda"), torch.randn(2, 1, S, 128, device="cuda")
    scaling = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=16)
    freqs = ops.rotary_frequencies(128, 256.0, axes=(16, 56, 56), scaling=scaling, interleaved=True, device="cuda")
    assert freqs.amplitude > 1
    a = angles(grid[None], freqs.inv_freq.tolist(), freqs.axis.tolist())
    for positions in (grid, grid[None].expand(2, -1, -1), grid.to(torch.int32), grid.t().contiguous().t()):
        for x, y in zip((q, k), ops.rotary(q, k, positions, freqs)):
            want = turn(x.double(), a, freqs.amplitude, True)
            close(y, want, rounding(torch.float32, want) + ROTATION * pair_size(x.double(), 64, freqs.amplitude, True))


def test_far_and_negative_positions_keep_their_angles():
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31 + 1, 2 ** 40 + 3, 0], device="cuda")
    x = torch.randn(1, 1, 4, 64, device="cuda")
    freqs = ops.rotary_frequencies(64, device="cuda")
    a = angles(pos[None, None], inverse_frequencies(64, 10000.0))
    want = turn(x.double(), a, 1.0, False)
    # 2^40 turns leave 2^-12 of 64 bits' 53; the product's rounding there is 2^40 2^-53 = 2^-13 of a radian on either side
    bound = 2 * a.abs().max(-1).values[:, None, :, None] * 2.0 ** -52
    y, _ = ops.rotary(x, None, pos, freqs)
    close(y, want, rounding(torch.float32, want) + (ROTATION + bound) * pair_size(x.double(), 32, 1.0, False))


def test_infinities_and_nan_stay_where_they_are():
    x = torch.randn(1, 2, 3, 16, device="cuda", dtype=torch.bfloat16)
    x[0, 0, 1, 12] = float("inf")
    x[0, 1, 2, 13] = float("nan")
    freqs = ops.rotary_frequencies(8, device="cuda")
    y, _ = ops.rotary(x, None, torch.arange(3, device="cuda"), freqs)
    assert torch.equal(torch.isfinite(y), torch.isfinite(x))
    assert torch.equal(y[..., 8:].nan_to_num(), x[..., 8:].nan_to_num())


def test_a_difference_of_the_forward_is_the_gradient():
    torch.manual_seed(3)
    q, k = (torch.randn(1, h, 9, 64, device="cuda", requires_grad=True) for h in (4, 2))
    w = [(1 + 0.2 * torch.randn(64, device="cuda")).requires_grad_() for _ in range(2)]
    freqs = ops.rotary_frequencies(32, device="cuda")
    pos = torch.arange(9, device="cuda")
    leaves = (q, k, *w)
    outs = ops.qk_norm_rotary(*leaves, pos, freqs)
    grads = [torch.randn_like(o) for o in outs]
    got = torch.autograd.grad(outs, leaves, grads)
    step = 2.0 ** -7
    for i, leaf in enumerate(leaves):
        d = torch.randn_like(leaf)
        d = d / d.norm()
        ends = []
        for s in (step, -step):
            moved = [t.detach() + (s * d if j == i else 0) for j, t in enumerate(leaves)]
            ends.append(sum((o.double() * g.double()).sum() for o, g in zip(ops.qk_norm_rotary(*moved, pos, freqs), grads)))
        along = float((got[i].double() * d.double()).sum())
        # rounding of the outputs over the step, and the third derivative: both far below one in a thousand of the gradient's size
        assert abs(float(ends[0] - ends[1]) / (2 * step) - along) <= 2e-3 * float(got[i].double().norm())


@pytest.mark.parametrize("tokens,heads_q,heads_k", [(0, 2, 1), (3, 0, 1), (3, 2, 0)])
def test_empty_operands(tokens, heads_q, heads_k):
    q = torch.randn(2, heads_q, tokens, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    k = torch.randn(2, heads_k, tokens, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    freqs = ops.rotary_frequencies(64, device="cuda")
    pos = torch.arange(tokens, device="cuda")
    for outs in (ops.rotary(q, k, pos, freqs), ops.qk_norm_rotary(q, k, w, w, pos, freqs)):
        assert [o.shape for o in outs] == [q.shape, k.shape]
        dq, dk = torch.autograd.grad(outs, (q, k), [torch.randn_like(o) for o in outs])
        assert bool(torch.isfinite(dq).all()) and bool(torch.isfinite(dk).all())


@pytest.mark.parametrize("tokens", [887, 888, 1184])
def test_tokens_on_either_side_of_whole_units(tokens):
    """A unit of work takes some heads of a token or all of them: the same results, and the same as of the tokens one by one."""
    torch.manual_seed(6)
    q, k = (torch.randn(1, tokens, h, 64, device="cuda", dtype=torch.bfloat16).transpose(1, 2).requires_grad_() for h in (20, 3))
    wq, wk = (torch.randn(64, device="cuda", dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    freqs, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(tokens, device="cuda")
    for op in (lambda a, b, p: ops.rotary(a, b, p, freqs), lambda a, b, p: ops.qk_norm_rotary(a, b, wq, wk, p, freqs)):
        out = op(q, k, pos)
        dout = [torch.randn_like(t) for t in out]
        grads = torch.autograd.grad(out, (q, k), dout)
        for i in range(0, tokens, 300):
            part = op(q[:, :, i:i + 300], k[:, :, i:i + 300], pos[i:i + 300])
            assert all(torch.equal(a, b[:, :, i:i + 300]) for a, b in zip(part, out))
            for a, b in zip(torch.autograd.grad(part, (q, k), [g[:, :, i:i + 300] for g in dout]), grads):
                assert torch.equal(a[:, :, i:i + 300], b[:, :, i:i + 300])


def test_norm_without_eps_at_heads_that_do_not_fill_a_warp():
    torch.manual_seed(5)
    q, k = (torch.randn(2, h, 9, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (3, 1))
    wq, wk = (torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(2))
    freqs, pos = ops.rotary_frequencies(64, device="cuda"), torch.arange(9, device="cuda")
    grads = []
    for eps in (0.0, 1e-12):        # which is nothing to squares of about 1
        out = ops.qk_norm_rotary(q, k, wq, wk, pos, freqs, eps=eps)
        grads.append(torch.autograd.grad(out, (q, k, wq, wk), [torch.ones_like(t) for t in out]))
    for a, b in zip(*grads):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


def test_only_what_needs_a_gradient_gets_one():
    freqs = ops.rotary_frequencies(64, device="cuda")
    pos = torch.arange(5, device="cuda")
    q, k = (torch.randn(1, 2, 5, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    k.requires_grad_()
    a, b = ops.rotary(q, k, pos, freqs)
    (a.float().sum() + b.float().sum()).backward()              # broadcast gradients of stride 0
    assert q.grad is None
    want, _ = ops.rotary(torch.ones_like(k), None, -pos, freqs)
    assert torch.equal(k.grad, want)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(ops.rotary(q, k, pos, freqs)[1].float().square().sum(), k, create_graph=True)
        g.float().sum().backward()


def test_streams_and_captured_graphs():
    torch.manual_seed(4)
    freqs = ops.rotary_frequencies(128, device="cuda")
    pos = torch.arange(50, device="cuda", dtype=torch.int32)
    q, k = torch.randn(2, 8, 50, 128, device="cuda", dtype=torch.bfloat16), torch.randn(2, 2, 50, 128, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(128, device="cuda", dtype=torch.bfloat16)
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        a, b, c, d = (t.detach().requires_grad_() for t in (q, k, w, w.clone()))
        outs = ops.qk_norm_rotary(a, b, c, d, pos, freqs)
        return (*[o.detach() for o in outs], *torch.autograd.grad(outs, (a, b, c, d), (gq, gk)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    q.copy_(torch.randn_like(q))
    pos.add_(1000)
    graph.replay()
    again = step()
    assert all(torch.equal(a, b) for a, b in zip(held, again))
    assert not torch.equal(held[0], want[0])


def test_wide_heads_take_the_plain_path_with_a_note():
    from teletron_b200.ops import fallback
    x = torch.randn(1, 1, 3, 320, device="cuda", dtype=torch.bfloat16)
    freqs = ops.rotary_frequencies(64, device="cuda")
    pos = torch.arange(3, device="cuda")
    n = sum(c for key, c in fallback.SEEN.items() if key.startswith("rotary"))
    was = fallback.strict()
    fallback.set_strict(False)
    try:
        y, _ = ops.rotary(x, None, pos, freqs)
        assert sum(c for key, c in fallback.SEEN.items() if key.startswith("rotary")) == n + 1 and y.shape == x.shape
        fallback.set_strict(True)
        with pytest.raises(fallback.LibraryFallbackError):
            ops.rotary(x, None, pos, freqs)
    finally:
        fallback.set_strict(was)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("behind", [1, 2])
@pytest.mark.parametrize("tokens", [1, 8, 100])
def test_gradients_at_other_alignments_than_the_inputs(tokens, behind, dtype):
    """What a concatenation's backward hands on: views into wider rows."""
    torch.manual_seed(7)
    q, k = (torch.randn(1, h, tokens, 128, device="cuda").to(dtype).requires_grad_() for h in (32, 8))
    w = [(1 + 0.2 * torch.randn(128, device="cuda")).to(dtype).requires_grad_() for _ in range(2)]
    freqs, pos = ops.rotary_frequencies(128, device="cuda"), torch.arange(tokens, device="cuda")
    a = angles(pos[None, None], inverse_frequencies(128, 10000.0))
    outs = ops.qk_norm_rotary(q, k, *w, pos, freqs)
    grads = [torch.randn(*o.shape[:3], 128 + behind, device="cuda").to(dtype)[..., behind:] for o in outs]
    got = torch.autograd.grad(outs, (q, k, *w), grads)
    rel = norm_error(128)
    for i, (x, g) in enumerate(zip((q, k), grads)):
        xd, wd, gd = x.detach().double(), w[i].detach().double(), g.double()
        r = torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-6)
        hat = xd * r
        back, back_size = turn(gd, -a, 1.0, False), pair_size(gd, 64, 1.0, False)
        dw = (back * hat).sum((0, 1, 2))
        close(got[2 + i], dw, rounding(dtype, dw) + (back_size * hat.abs()).sum((0, 1, 2)) * (x[..., 0].numel() * U32 + ROTATION + rel), "dw")
        gw = back * wd
        dx = r * (gw - hat * (gw * hat).mean(-1, keepdim=True))
        spread = r * (back_size * wd.abs() + hat.abs() * (back_size * wd.abs() * hat.abs()).mean(-1, keepdim=True))
        close(got[i], dx, rounding(dtype, dx) + spread * (ROTATION + 3 * rel + 128 * U32), "dx")
