"""``ops.rotary`` and ``ops.qk_norm_rotary`` without a GPU: frequencies, the plain path, gradients, refusals."""

import math

import pytest
import torch

from rotary_oracle import angles, inverse_frequencies, turn
from teletron_b200 import ops


def test_frequencies_follow_the_published_scalings():
    dim, theta = 64, 10000.0
    base = torch.tensor(inverse_frequencies(dim, theta), dtype=torch.float64)
    plain = ops.rotary_frequencies(dim, theta)
    assert torch.allclose(plain.inv_freq, base, rtol=1e-14, atol=0) and plain.amplitude == 1.0 and plain.dim == dim
    assert torch.allclose(ops.rotary_frequencies(dim, theta, scaling={"rope_type": "linear", "factor": 4}).inv_freq, base / 4, rtol=1e-14)
    ntk = ops.rotary_frequencies(dim, theta, scaling={"rope_type": "ntk", "factor": 4.0}).inv_freq
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(base[-1]) / 4, rel_tol=1e-12)       # the slowest pair is stretched by the factor
    ll = ops.rotary_frequencies(dim, theta, scaling=dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                         original_max_position_embeddings=8192)).inv_freq
    wave = 2 * math.pi / base
    assert torch.allclose(ll[wave < 8192 / 4], base[wave < 8192 / 4], rtol=1e-14)
    assert torch.allclose(ll[wave > 8192], base[wave > 8192] / 8, rtol=1e-14)
    between = (wave >= 8192 / 4) & (wave <= 8192)
    assert bool(between.any()) and bool((ll[between] <= base[between]).all()) and bool((ll[between] >= base[between] / 8).all())
    yarn = ops.rotary_frequencies(dim, theta, scaling=dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096))
    assert math.isclose(yarn.amplitude, 0.1 * math.log(4) + 1) and yarn.inv_freq[0] == 1.0
    assert math.isclose(float(yarn.inv_freq[-1]), float(base[-1]) / 4, rel_tol=1e-12)


def test_frequencies_equal_the_installed_models():
    """The same dictionaries through the text encoders' own package."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    for kind, extra in (("linear", {}), ("llama3", dict(low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=2048)),
                        ("yarn", dict(original_max_position_embeddings=2048))):
        scaling = dict(rope_type=kind, factor=4.0, rope_theta=500000.0, **extra)
        cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=8192, rope_parameters=scaling)
        inv, amplitude = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu")
        mine = ops.rotary_frequencies(128, 500000.0, scaling=scaling)
        assert torch.allclose(mine.inv_freq.float(), inv.float(), rtol=1e-5, atol=0), kind
        assert math.isclose(mine.amplitude, amplitude, rel_tol=1e-6)


def test_axes_restate_the_video_table():
    from teletron_b200.models.hunyuanvideo.embeddings import HunyuanVideoRotaryPosEmbed
    cos, sin = HunyuanVideoRotaryPosEmbed(2, 1, (16, 56, 56), 256.0)(torch.zeros(1, 16, 3, 8, 10))
    grid = torch.stack([t.reshape(-1) for t in torch.meshgrid(torch.arange(3), torch.arange(4), torch.arange(5), indexing="ij")])
    x = torch.randn(1, 2, 60, 128)
    freqs = ops.rotary_frequencies(128, 256.0, axes=(16, 56, 56), interleaved=True)
    got, none = ops.rotary(x, None, grid, freqs)
    assert none is None
    # the table's angles are fp32: at most 2^-24 relative, times positions below 5
    assert torch.allclose(got, ops.apply_rope(x, cos, sin), atol=1e-5, rtol=0)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(16, 16), (20, 10), (8, 2)])
def test_plain_path_against_complex_multiplication(interleaved, dim, rot):
    torch.manual_seed(0)
    q, k = torch.randn(2, 3, 5, dim, dtype=torch.float64), torch.randn(2, 1, 5, dim, dtype=torch.float64)
    pos = torch.tensor([[0, 1, 2, 3, 4], [100000, 100001, 7, 7, -3]])
    freqs = ops.rotary_frequencies(rot, 10000.0, interleaved=interleaved)
    a = angles(pos[:, None], inverse_frequencies(rot, 10000.0))
    for got, x in zip(ops.rotary(q, k, pos, freqs), (q, k)):
        assert torch.allclose(got, turn(x, a, 1.0, interleaved), rtol=0, atol=1e-9)
        assert torch.equal(got[..., rot:], x[..., rot:])


def test_gradients_against_differences():
    torch.manual_seed(1)
    freqs = ops.rotary_frequencies(6, 50.0)
    pos = torch.tensor([3, 9, 0])
    q, k = (torch.randn(2, h, 3, 8, dtype=torch.float64, requires_grad=True) for h in (2, 1))
    w = [torch.randn(8, dtype=torch.float64, requires_grad=True) for _ in range(2)]
    assert torch.autograd.gradcheck(lambda a, b: ops.rotary(a, b, pos, freqs), (q, k))
    assert torch.autograd.gradcheck(lambda a, b, c, d: ops.qk_norm_rotary(a, b, c, d, pos, freqs), (q, k, *w))


def test_norm_is_the_ops_rmsnorm():
    torch.manual_seed(2)
    q, w = torch.randn(1, 2, 4, 16), torch.randn(16)
    freqs = ops.rotary_frequencies(16)
    pos = torch.arange(4)
    got, _ = ops.qk_norm_rotary(q, q, w, w, pos, freqs, eps=1e-3)
    assert torch.allclose(got, ops.rotary(ops.rmsnorm(q, w, 1e-3), None, pos, freqs)[0], atol=1e-6)


@pytest.mark.parametrize("kw", [dict(dim=7), dict(dim=0), dict(dim=8, axes=(4, 2)), dict(dim=8, axes=(5, 3)), dict(dim=8, theta=0.0),
                                dict(dim=8, theta=float("inf")), dict(dim=8, scaling={"rope_type": "spiral", "factor": 2}),
                                dict(dim=8, scaling={"rope_type": "linear"}), dict(dim=8, scaling={"rope_type": "linear", "factor": 0}),
                                dict(dim=8, scaling={"rope_type": "linear", "factor": float("nan")}), dict(dim=2, scaling={"rope_type": "ntk", "factor": 2}),
                                dict(dim=8, scaling=dict(rope_type="llama3", factor=8, low_freq_factor=4, high_freq_factor=1,
                                                         original_max_position_embeddings=64)),
                                dict(dim=8, theta=1.0, scaling=dict(rope_type="yarn", factor=8, original_max_position_embeddings=64))])
def test_frequencies_refuse(kw):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(**kw)


def _operands():
    return dict(q=torch.randn(2, 3, 4, 8), k=torch.randn(2, 1, 4, 8), positions=torch.arange(4), freqs=ops.rotary_frequencies(8))


@pytest.mark.parametrize("change", [dict(q=torch.randn(3, 4, 8)), dict(k=torch.randn(2, 1, 5, 8)), dict(k=torch.randn(1, 1, 4, 8)),
                                    dict(k=torch.randn(2, 1, 4, 8).half()), dict(positions=torch.arange(4.0)), dict(positions=torch.arange(5)),
                                    dict(positions=torch.zeros(3, 4, dtype=torch.long)), dict(positions=torch.zeros(2, 1, 4, dtype=torch.int16)),
                                    dict(freqs=ops.rotary_frequencies(10)), dict(freqs=ops.rotary_frequencies(8, axes=(4, 4))), dict(freqs=None),
                                    dict(q=torch.zeros(2, 3, 4, 8, dtype=torch.int32), k=None)])
def test_operands_that_do_not_belong_together_are_refused(change):
    with pytest.raises(ValueError):
        ops.rotary(**{**_operands(), **change})


@pytest.mark.parametrize("shape,dtype", [((7,), torch.float32), ((1, 8), torch.float32), ((8,), torch.bfloat16)])
def test_norm_weights_are_checked(shape, dtype):
    a = _operands()
    good = torch.ones(8)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(a["q"], a["k"], torch.ones(shape, dtype=dtype), good, a["positions"], a["freqs"])
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(a["q"], a["k"], good, torch.ones(shape, dtype=dtype), a["positions"], a["freqs"])


@pytest.mark.parametrize("eps", [-1e-6, float("nan"), float("inf")])
def test_eps_is_checked(eps):
    a, w = _operands(), torch.ones(8)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(a["q"], a["k"], w, w, a["positions"], a["freqs"], eps=eps)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(a["q"], None, w, w, a["positions"], a["freqs"])


@pytest.mark.parametrize("change", [dict(half_turns=torch.ones(3, dtype=torch.float64)), dict(half_turns=torch.ones(4)),
                                    dict(axis=torch.zeros(4, dtype=torch.int64)), dict(axis=torch.zeros(8, dtype=torch.int32)[::2]),
                                    dict(half_turns=torch.ones(8, dtype=torch.float64)[::2])])
def test_frequencies_of_other_shapes_are_refused(change):
    import dataclasses
    with pytest.raises(ValueError):
        dataclasses.replace(ops.rotary_frequencies(8), **change)


def test_native_arguments_have_the_layout_that_the_library_expects():
    """The packed arguments are read as the C structure; sizes that disagree are refused before anything is launched."""
    from teletron_b200.ops import _lib, rope
    if not _lib.available():
        pytest.skip("native library not built")
    ok = rope._ARGS.pack(rope._ARGS.size, 1, 4, 2, 1, 8, 4, 2, 0, 0, 0, 16, 16, *[0] * 6, 16, 16, *[0] * 6, 16, 0, 0, 1, 16, 0, 1.0, 0.0,
                         16, 16, 16, 16, *[0] * 6, 16, 16, 0, 0)
    assert _lib.lib().tt_rotary_partial_floats(ok) > 0
    assert _lib.lib().tt_rotary_partial_floats(b"\x08" + ok[1:]) == -1
    wide = rope._ARGS.pack(rope._ARGS.size, 1, 4, 2, 1, 258, 4, 2, 0, 0, 0, 16, 16, *[0] * 6, 16, 16, *[0] * 6, 16, 0, 0, 1, 16, 0, 1.0, 0.0,
                           16, 16, 16, 16, *[0] * 6, 16, 16, 0, 0)
    assert _lib.lib().tt_norm_rotary_fwd(wide, None) == 4


def _recorded(monkeypatch):
    """The native calls of the op layer, noted instead of made, on tensors of the host."""
    import contextlib
    from teletron_b200.ops import rope
    calls = []
    monkeypatch.setattr(rope, "call", lambda name, args, stream: calls.append((name, args)))
    monkeypatch.setattr(rope, "stream", lambda: None)
    monkeypatch.setattr(rope, "on_device", lambda t: contextlib.nullcontext())
    return calls


@pytest.mark.parametrize("tokens", [1, 8, 100, 887, 2000])
@pytest.mark.parametrize("behind", [0, 1, 2])
def test_the_scratch_of_the_norms_backward_is_sized_for_its_gradients(monkeypatch, tokens, behind):
    """Gradients at other alignments than the inputs (views into wider rows) change how the work is shared out."""
    from teletron_b200.ops import _lib, rope
    if not _lib.available():
        pytest.skip("native library not built")
    calls = _recorded(monkeypatch)
    q, k = (torch.randn(1, h, tokens, 128).bfloat16().requires_grad_() for h in (32, 8))
    w = torch.ones(128, dtype=torch.bfloat16, requires_grad=True)
    outs = rope.qk_norm_rotary(q, k, w, w, torch.arange(tokens), (0, 0, 1), ops.rotary_frequencies(128), 1e-6)
    torch.autograd.grad(outs, (q, k), [torch.randn(1, h, tokens, 128 + behind).bfloat16()[..., behind:] for h in (32, 8)])
    (name, args), = calls[1:]
    assert name == "tt_norm_rotary_bwd"
    given, = rope.struct.unpack_from("@l", args, len(args) - 8)
    assert given == _lib.lib().tt_rotary_partial_floats(args) > 0


@pytest.mark.parametrize("extra", [dict(truncate=False), dict(truncate=True), dict(truncate=False, beta_fast=20.0, beta_slow=2.0),
                                   dict(mscale=0.707, mscale_all_dim=0.707), dict(mscale=1.0, mscale_all_dim=0.707), dict(mscale=1.0, mscale_all_dim=0.5),
                                   dict(mscale=0.5), dict(mscale_all_dim=0.5), dict(mscale=1.0, mscale_all_dim=0.0), dict(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.25),
                                   dict(attention_factor=None, mscale=None, mscale_all_dim=None, beta_fast=None, truncate=True)])
@pytest.mark.parametrize("factor", [4.0, 40.0, 1.0])
def test_yarn_follows_all_of_its_keys(extra, factor):
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    scaling = dict(rope_type="yarn", factor=factor, rope_theta=500000.0, original_max_position_embeddings=2048, **extra)
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, max_position_embeddings=8192, rope_parameters=dict(scaling))
    inv, amplitude = ROPE_INIT_FUNCTIONS["yarn"](cfg, "cpu")
    mine = ops.rotary_frequencies(128, 500000.0, scaling=scaling)
    assert torch.allclose(mine.inv_freq.float(), inv.float(), rtol=1e-5, atol=0)
    assert math.isclose(mine.amplitude, amplitude, rel_tol=1e-6)


def test_yarn_without_truncation_and_with_two_scales_by_its_formulas():
    dim, theta, factor, context = 64, 10000.0, 8.0, 4096
    got = ops.rotary_frequencies(dim, theta, scaling=dict(rope_type="yarn", factor=factor, original_max_position_embeddings=context, truncate=False,
                                                          mscale=1.2, mscale_all_dim=0.4))
    assert math.isclose(got.amplitude, (0.12 * math.log(factor) + 1) / (0.04 * math.log(factor) + 1), rel_tol=1e-12)
    low, high = (dim * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (32, 1))
    for j, (have, base) in enumerate(zip(got.inv_freq.tolist(), inverse_frequencies(dim, theta))):
        stretched = min(max((j - low) / (high - low), 0.0), 1.0)
        assert math.isclose(have, base * (1 - stretched) + base / factor * stretched, rel_tol=1e-12)


@pytest.mark.parametrize("scaling", [dict(rope_type="linear", factor=2.0, short_factor=[1.0]), dict(rope_type="default", alpha=3.0), dict(factor=4.0),
                                     dict(rope_type="linear", factor=None), dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, mscal=1.0),
                                     dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, attention_factor=float("nan")),
                                     dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, attention_factor=1e300),
                                     dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, mscale=float("inf"), mscale_all_dim=1.0),
                                     dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, mscale=1.0, mscale_all_dim=-10 / math.log(4.0)),
                                     dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64, beta_fast=-1.0),
                                     dict(rope_type="linear", factor=4.0, rope_theta=500000.0)])
def test_scalings_that_would_not_be_followed_are_refused(scaling):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(128, 10000.0, scaling=scaling)


def test_what_configurations_hold_beside_the_scaling_is_taken():
    plain = ops.rotary_frequencies(128, 500000.0)
    for scaling in ({}, dict(rope_type="default", rope_theta=500000.0), dict(type="default", partial_rotary_factor=0.5), dict(rope_type="default", factor=None),
                    dict(rope_type="default", factor=1.0, original_max_position_embeddings=8192), dict(rope_theta=500000.0),
                    dict(rope_type="linear", factor=1.0, finetuned=True, max_position_embeddings=8192), dict(rope_type=None, type="linear", factor=1.0)):
        got = ops.rotary_frequencies(128, 500000.0, scaling=scaling)
        assert torch.equal(got.inv_freq, plain.inv_freq) and got.amplitude == 1.0


def test_forward_mode_derivatives_are_refused_not_lost(monkeypatch):
    """Dual tensors need no ``requires_grad``; a kernel reads their primals alone."""
    import torch.autograd.forward_ad as fwd
    from teletron_b200.ops import _lib, rope
    if not _lib.available():
        pytest.skip("native library not built")
    calls = _recorded(monkeypatch)
    freqs, pos, w = ops.rotary_frequencies(64), torch.arange(3), torch.ones(64)
    q, k = torch.randn(1, 2, 3, 64), torch.randn(1, 1, 3, 64)
    with fwd.dual_level():
        for grad in (True, False):
            for which in range(4):
                args = [q, k, w, w]
                args[which] = fwd.make_dual(args[which], torch.ones_like(args[which]))
                with torch.set_grad_enabled(grad):
                    with pytest.raises(RuntimeError):
                        rope.qk_norm_rotary(*args, pos, (0, 0, 1), freqs, 1e-6)
                    if which < 2:
                        with pytest.raises(RuntimeError):
                            rope.rotary(*args[:2], pos, (0, 0, 1), freqs)
        with pytest.raises(RuntimeError):
            rope.rotary(fwd.make_dual(q, q), None, pos, (0, 0, 1), freqs)
        n = len(calls)
        rope.rotary(q, k, pos, (0, 0, 1), freqs)            # no tangents: as ever
        rope.qk_norm_rotary(q, k, w, w, pos, (0, 0, 1), freqs, 1e-6)
        assert len(calls) == n + 2
        # the plain path carries them
        out, _ = ops.rotary(fwd.make_dual(q, q), None, pos, freqs)
        assert torch.allclose(fwd.unpack_dual(out).tangent, ops.rotary(q, None, pos, freqs)[0], atol=1e-5)
    with pytest.raises(RuntimeError):           # the same by transformation
        torch.func.jvp(lambda x: rope.rotary(x, k, pos, (0, 0, 1), freqs)[0], (q,), (q,))
