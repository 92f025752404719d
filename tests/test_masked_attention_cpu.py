"""``ops.key_ranges`` and ``ops.masked_attention`` without a GPU: runs, the plain path, gradients, refusals."""

import ctypes

import pytest
import torch

from attention_oracle import runs
from teletron_b200 import ops

CASES = [dict(q_len=7), dict(q_len=7, causal=True), dict(q_len=5, kv_len=9), dict(q_len=3, kv_len=8, causal=True, query_start=4),
         dict(q_len=9, causal=True, prefix_len=4), dict(q_len=9, batch=2, causal=True, prefix_len=[0, 30]),
         dict(q_len=12, documents=[0, 4, 4, 9]), dict(q_len=12, batch=2, documents=[[0, 12], [3, 5]]),
         dict(q_len=12, batch=2, causal=True, documents=[[0, 5, 12], [2, 6, 7]], prefix_len=[[2, 0], [9, 1]]),
         dict(q_len=12, batch=2, causal=True, documents=[[0, 5, 12], [2, 6, 7]], prefix_len=[3, 1]),
         dict(q_len=6, batch=3, kv_valid_len=[0, 1, 6]), dict(q_len=2, kv_len=10, batch=3, causal=True, kv_valid_len=[10, 3, 0], query_start=[8, 1, -1]),
         dict(q_len=1, kv_len=1), dict(q_len=4, kv_valid_len=99), dict(q_len=4, kv_valid_len=-3), dict(q_len=130, causal=True, documents=[0, 129])]


def expected(kw):
    a = dict(kw)
    B, n = a.pop("batch", 1), a.pop("q_len")
    m = a.pop("kv_len", n)
    return runs(n, m, B, a.get("causal", False), a.get("documents"), a.get("prefix_len", 0), a.get("kv_valid_len"), a.get("query_start", 0))


@pytest.mark.parametrize("kw", CASES)
def test_runs_are_the_definitions(kw):
    got = ops.key_ranges(**kw)
    first, behind = expected(kw)
    assert torch.equal(got.first, first) and torch.equal(got.behind, behind)


@pytest.mark.parametrize("kw", [dict(q_len=-1), dict(q_len=3, kv_len=-1), dict(q_len=3, batch=-1), dict(q_len=3, prefix_len=1), dict(q_len=3, kv_len=4, causal=True),
                                dict(q_len=3, kv_len=4, documents=[0, 3]), dict(q_len=3, documents=[0, 3], query_start=1), dict(q_len=3, documents=[0]),
                                dict(q_len=3, documents=torch.tensor([0.0, 3.0])), dict(q_len=3, batch=2, documents=[[0, 3]]),
                                dict(q_len=3, causal=True, prefix_len=-1), dict(q_len=3, batch=2, causal=True, prefix_len=[1]),
                                dict(q_len=3, batch=2, causal=True, prefix_len=[[1, 2], [1, 2]]), dict(q_len=3, batch=2, kv_valid_len=[1, 2, 3]),
                                dict(q_len=3, batch=2, kv_valid_len=torch.tensor([1.0, 2.0])), dict(q_len=3, batch=2, query_start=torch.zeros(2, 1, dtype=torch.int32))])
def test_key_ranges_refuses(kw):
    with pytest.raises(ValueError):
        ops.key_ranges(**kw)


def test_lengths_beyond_32_bits():
    huge, n = 2 ** 32 + 1, 6
    want = ops.key_ranges(n, batch=2, causal=True, prefix_len=n, kv_valid_len=n)
    for kw in (dict(prefix_len=huge), dict(prefix_len=[huge, huge]), dict(query_start=huge), dict(query_start=torch.tensor([huge, huge])),
               dict(prefix_len=n, kv_valid_len=huge), dict(prefix_len=n, kv_valid_len=[huge, huge]), dict(prefix_len=n, documents=[0, huge])):
        got = ops.key_ranges(n, batch=2, causal=True, **kw)
        assert torch.equal(got.first, want.first) and torch.equal(got.behind, want.behind), kw
    none = ops.key_ranges(n, batch=2, causal=True, query_start=-huge)
    assert not bool(none.behind.any())
    with pytest.raises(ValueError):
        ops.key_ranges(huge)


def _operands(**change):
    a = dict(q=torch.randn(2, 4, 6, 8), k=torch.randn(2, 2, 6, 8), v=torch.randn(2, 2, 6, 8), ranges=ops.key_ranges(6, batch=2))
    a.update(change)
    return a


@pytest.mark.parametrize("change", [dict(q=torch.randn(2, 4, 8)), dict(k=torch.randn(2, 3, 6, 8), v=torch.randn(2, 3, 6, 8)), dict(k=torch.randn(2, 2, 5, 8)),
                                    dict(v=torch.randn(2, 2, 6, 8).half()), dict(q=torch.randn(1, 4, 6, 8)), dict(ranges=None), dict(ranges=ops.key_ranges(6)),
                                    dict(ranges=ops.key_ranges(5, 6, batch=2)), dict(scale=float("nan")), dict(scale=1e300), dict(softcap=1e-300),
                                    dict(softcap=1e38), dict(softcap=float("nan")), dict(scale=1e20, softcap=1e-20), dict(softcap=0.0), dict(softcap=-1.0),
                                    dict(softcap=float("inf")), dict(distance_bias=torch.zeros(4, 4)), dict(distance_bias=torch.zeros(2, 5)),
                                    dict(distance_bias=torch.zeros(4, 5).double()), dict(distance_bias=torch.zeros(5)),
                                    dict(q=torch.zeros(2, 4, 6, 8, dtype=torch.int32), k=torch.zeros(2, 2, 6, 8, dtype=torch.int32), v=torch.zeros(2, 2, 6, 8, dtype=torch.int32))])
def test_masked_attention_refuses(change):
    with pytest.raises(ValueError):
        ops.masked_attention(**_operands(**change))


def test_plain_path_is_softmax_attention():
    torch.manual_seed(0)
    q, k, v = (torch.randn(2, h, 9, 16, dtype=torch.float64) for h in (4, 2, 2))
    kk, vv = k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)
    import torch.nn.functional as F
    want = F.scaled_dot_product_attention(q, kk, vv, is_causal=True).transpose(1, 2).reshape(2, 9, 64)
    assert torch.allclose(ops.masked_attention(q, k, v, ops.key_ranges(9, batch=2, causal=True)), want, atol=1e-12)
    assert torch.allclose(ops.masked_attention(q, kk, vv, ops.key_ranges(9, batch=2)), ops.attention(q, kk, vv), atol=1e-12)


def test_rows_and_keys_without_a_run_are_left_out():
    torch.manual_seed(1)
    q, k, v = (torch.randn(1, 2, 8, 4, dtype=torch.float64) for _ in range(3))
    r = ops.key_ranges(8, documents=[1, 6])
    want = ops.masked_attention(q, k, v, r)
    for t in (q, k, v):
        t[:, :, [0, 6, 7]] = float("nan")
    got = ops.masked_attention(q, k, v, r)
    assert torch.equal(got, want) and not bool(got[:, [0, 6, 7]].any())
    # nor do they reach a gradient, or the other way
    dout = torch.randn(1, 8, 8, dtype=torch.float64)
    dout[:, [0, 6, 7]] = float("inf")
    for g in torch.autograd.grad(ops.masked_attention(*[t.requires_grad_() for t in (q, k, v)], r, softcap=3.0), (q, k, v), dout):
        assert bool(torch.isfinite(g).all()) and not bool(g[:, :, [0, 6, 7]].any())


def test_gradients_against_differences():
    torch.manual_seed(2)
    q, k, v = (torch.randn(2, h, 5, 4, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2))
    bias = torch.randn(4, 5, requires_grad=True)
    r = ops.key_ranges(5, batch=2, causal=True, documents=[[0, 3, 5], [0, 4, 4]], prefix_len=2)
    assert torch.autograd.gradcheck(lambda a, b, c: ops.masked_attention(a, b, c, r, softcap=2.0, distance_bias=bias.detach()), (q, k, v))
    # the table is fp32: its gradient against differences of 2^-6, whose own error is their square times the third derivative
    w = torch.randn(2, 5, 16, dtype=torch.float64)
    g, = torch.autograd.grad((ops.masked_attention(q, k, v, r, distance_bias=bias) * w).sum(), bias)
    d = torch.randn(4, 5)
    step = 2.0 ** -6
    ends = [(ops.masked_attention(q, k, v, r, distance_bias=bias.detach() + s * d) * w).sum() for s in (step, -step)]
    assert abs(float((ends[0] - ends[1]).detach()) / (2 * step) - float((g * d).sum())) < 1e-2 * float(g.norm() * d.norm())


def test_empty_operands():
    for B, n, m in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        q, k = torch.randn(B, 2, n, 4), torch.randn(B, 2, m, 4)
        out = ops.masked_attention(q, k, k, ops.key_ranges(n, m, batch=B))
        assert out.shape == (B, n, 8) and not bool(out.any() and m == 0)


def _native():
    from teletron_b200.ops import _lib
    if not _lib.available():
        pytest.skip("native library not built")
    return _lib.lib()


def test_native_arguments_are_checked_ahead_of_any_launch():
    lib = _native()
    from teletron_b200.ops import attn_ranges as A
    fields = dict(size=A._ARGS.size, batch=1, q_heads=4, k_heads=2, q_len=8, kv_len=8, head_dim=64, dtype=0, distance=-1)

    def pack(scale=1.0, softcap=0.0, plan=256, bias=0, dout=0, **kw):
        f = {**fields, **kw}
        return A._ARGS.pack(f["size"], f["batch"], f["q_heads"], f["k_heads"], f["q_len"], f["kv_len"], f["head_dim"], f["dtype"], f["distance"], 0, 0,
                            256, 256, 256, *[64] * 9, 256, 0, 256, plan, bias, scale, softcap, dout, 0, 0, 0, 0, *[0] * 9, 0, 0, 256)

    for kw, code in ((dict(size=8), 1), (dict(batch=0), 1), (dict(batch=65536), 1), (dict(k_heads=3), 1), (dict(q_len=0), 1), (dict(kv_len=2 ** 30 + 1), 1),
                     (dict(head_dim=96), 4), (dict(dtype=2), 1), (dict(distance=5), 1), (dict(distance=1025, bias=256), 4), (dict(bias=256), 1),
                     (dict(scale=float("nan")), 1), (dict(softcap=-1.0), 1), (dict(softcap=float("inf")), 1), (dict(plan=0), 1), (dict(plan=8), 1)):
        assert lib.tt_attn_ranges_fwd(pack(**kw), None) == code, kw
        assert lib.tt_attn_ranges_bwd(pack(**kw), None) == code, kw
    assert lib.tt_attn_ranges_bwd(pack(), None) == 1            # nothing to differentiate


def test_plan_parts_do_not_overlap():
    from teletron_b200.ops import attn_ranges as A
    _native()
    for B, n, m in ((1, 1, 1), (3, 129, 127), (2, 1, 70000)):
        at = A._layout(B, n, m)
        qt, kt = -(-n // 128), -(-m // 128)
        sizes = [("q_tiles", 4 * B * qt), ("dead", 4 * B * kt), ("k_tiles", 2 * B * kt), ("dirty", B * kt), ("first", B * n), ("behind", B * n), ("start", B)]
        place = 0
        for name, size in sizes:
            assert getattr(at, name) == place
            place += size
        assert at.ints == place and at.dead % 4 == 0 and at.k_tiles % 2 == 0
    assert isinstance(ctypes.sizeof(A._Layout), int)


def test_forward_mode_derivatives_are_refused_not_lost(monkeypatch):
    """Dual tensors need no ``requires_grad``; a kernel reads their primals alone."""
    import contextlib
    import torch.autograd.forward_ad as fwd
    from teletron_b200.ops import _lib, attn_ranges
    if not _lib.available():
        pytest.skip("native library not built")
    calls = []
    monkeypatch.setattr(attn_ranges, "call", lambda name, *args: calls.append(name))
    monkeypatch.setattr(attn_ranges, "stream", lambda: None)
    monkeypatch.setattr(attn_ranges, "on_device", lambda t: contextlib.nullcontext())
    n, m = 40, 200
    ranges = ops.key_ranges(n, m, batch=2)
    object.__setattr__(ranges, "plan", torch.zeros(16, dtype=torch.int32))
    q, k, v = (torch.randn(2, h, s, 64).bfloat16() for h, s in ((4, n), (2, m), (2, m)))
    bias = torch.randn(4, 5)
    with fwd.dual_level():
        for grad in (True, False):
            for which in range(4):
                args = [q, k, v, bias]
                args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    attn_ranges.masked_attention(*args[:3], ranges, None, None, args[3])
        before = len(calls)
        attn_ranges.masked_attention(q, k, v, ranges, None, None, bias)         # no tangents: as ever
        assert len(calls) == before + 1
    with pytest.raises(RuntimeError):           # the same by transformation
        torch.func.jvp(lambda x: attn_ranges.masked_attention(x, k, v, ranges, None, None, None), (q,), (q,))
