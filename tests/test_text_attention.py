"""The text encoders on this package's rotation and attention against the same weights on their library's."""

import copy

import pytest
import torch

from teletron_b200.models.text_attention import distance_buckets, prompt_ranges, use_native_attention
from teletron_b200.models.text_encoders import LlamaTextEncoder, PromptEncoder, clip_text_config, llama_config, t5_config

PROMPTS = ["a short prompt", "another slightly longer prompt here with words", "x"]


def _llama(**kw):
    torch.manual_seed(0)
    cfg = llama_config(3, 64, 4, 2, 128, 1000)
    return cfg, LlamaTextEncoder(max_length=24, dtype=torch.float32, config=cfg, **kw)


@pytest.mark.parametrize("scaling", [None, dict(rope_type="llama3", factor=4.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                                original_max_position_embeddings=16, rope_theta=500000.0)])
def test_llama_states_equal_the_librarys(scaling):
    torch.manual_seed(0)
    cfg = llama_config(3, 64, 4, 2, 128, 1000)
    if scaling is not None:
        cfg.rope_parameters = scaling
    plain = LlamaTextEncoder(max_length=24, dtype=torch.float32, config=cfg)
    native = copy.deepcopy(plain)
    native.native = use_native_attention(native.model)
    want, mask = plain(PROMPTS)
    got, got_mask = native(PROMPTS)
    assert torch.equal(mask, got_mask)
    # fp32 throughout: three layers of products over at most 128 terms, states of the order of 1
    assert torch.allclose(got, want, atol=2e-4, rtol=0)
    # a prompt by itself, not padded
    assert torch.allclose(native(PROMPTS[:1])[0][:, :4], want[:1, :4], atol=2e-4, rtol=0)


def test_t5_states_equal_the_librarys():
    torch.manual_seed(1)
    plain = PromptEncoder("t5", max_length=200, dtype=torch.float32, configs=[t5_config(2, 32, 4, 64, 300)])
    plain.load_model()
    native = copy.deepcopy(plain)
    native.encoders[0].native = use_native_attention(native.encoders[0].model)
    for p in (plain, native):           # a table whose entries differ
        w = p.encoders[0].model.encoder.block[0].layer[0].SelfAttention.relative_attention_bias.weight
        w.copy_(torch.linspace(-2, 2, w.numel()).view_as(w))
    for with_mask in (False, True):
        want, mask = plain(PROMPTS, with_attention_mask=with_mask)
        got, _ = native(PROMPTS, with_attention_mask=with_mask)
        assert torch.allclose(got, want, atol=2e-4, rtol=0)


def test_buckets_are_the_librarys():
    from transformers.models.t5.modeling_t5 import T5Attention
    for R, n, both in ((128, 32, True), (64, 16, True), (128, 32, False), (20, 8, False)):
        d = torch.arange(-R, R + 1)
        want = T5Attention._relative_position_bucket(d, bidirectional=both, num_buckets=n, max_distance=R)
        assert torch.equal(distance_buckets(R, n, both), want)


def test_prompts_padded_on_either_side():
    right = torch.tensor([[1, 1, 0, 0], [1, 1, 1, 1]])
    r = prompt_ranges(right, 2, 4, True, "cpu")
    assert r.behind.tolist() == [[1, 2, 2, 2], [1, 2, 3, 4]] and not bool(r.first.any())
    r = prompt_ranges(right.flip(1), 2, 4, True, "cpu")
    assert r.first.tolist() == [[0, 0, 2, 2], [0, 0, 0, 0]] and r.behind.tolist() == [[0, 0, 3, 4], [1, 2, 3, 4]]
    with pytest.raises(ValueError):
        prompt_ranges(torch.tensor([[1, 0, 1, 0]]), 1, 4, True, "cpu")


def test_refusals_and_flag():
    with pytest.raises(ValueError):
        PromptEncoder("clip_text", native_attention=True)
    with pytest.raises(ValueError):
        use_native_attention(torch.nn.Linear(2, 2))
    cfg, enc = _llama(native_attention=True)
    assert enc.native is not None and _llama()[1].native is None
    emb, mask = PromptEncoder("llama", max_length=10, dtype=torch.float32, configs=[cfg], native_attention=True)(PROMPTS, with_attention_mask=True)
    assert emb.shape == (3, 10, 64) and mask.shape == (3, 10)
    from teletron_b200.training.args import parse_args
    assert parse_args(argv=["--encoder-native-attention"]).encoder_native_attention is True
    assert clip_text_config() is not None


class _Config:
    """A configuration as the encoders' package had it ahead of its release 5: the scaling apart from the base."""

    def __init__(self, rope_scaling, rope_theta=500000.0, **kw):
        self.hidden_size, self.num_attention_heads, self.rope_scaling, self.rope_theta = 64, 4, rope_scaling, rope_theta
        self.__dict__.update(kw)


@pytest.mark.parametrize("scaling", [None, dict(rope_type="llama3", factor=4.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=16),
                                     dict(type="linear", factor=3.0)])
def test_scalings_of_older_configurations_are_followed(scaling):
    from teletron_b200 import ops
    from teletron_b200.models.text_attention import rotary_of
    for kw, dim in ((dict(), 16), (dict(partial_rotary_factor=0.5), 8), (dict(head_dim=32), 32)):
        got, want = rotary_of(_Config(scaling, **kw)), ops.rotary_frequencies(dim, 500000.0, scaling=scaling)
        assert torch.equal(got.inv_freq, want.inv_freq) and got.amplitude == want.amplitude
    now = rotary_of(_Config(dict(rope_type="linear", factor=3.0), rope_parameters=dict(rope_type="linear", factor=5.0, rope_theta=10000.0)))
    assert torch.equal(now.inv_freq, ops.rotary_frequencies(16, 10000.0, scaling=dict(rope_type="linear", factor=5.0)).inv_freq)


def test_a_model_that_rotates_otherwise_than_its_configuration_says_is_refused():
    """Frequencies from the configuration are compared with the model's own, whatever names a release keeps them under."""
    enc = _llama()[1]
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        use_native_attention(copy.deepcopy(enc.model).to(dtype))
    enc.model.rotary_emb.inv_freq.div_(4.0)
    with pytest.raises(ValueError):
        use_native_attention(enc.model)
    enc = _llama()[1]
    enc.model.rotary_emb.attention_scaling = 1.2
    with pytest.raises(ValueError):
        use_native_attention(enc.model)
    assert type(enc.model.layers[0].self_attn).__name__ == "LlamaAttention"         # as it was


@pytest.mark.parametrize("kind", ["llama", "t5"])
def test_two_threads_on_one_encoder_keep_their_own_masks(kind):
    import threading
    if kind == "llama":
        enc = _llama(native_attention=True)[1]
        model, call = enc.model, lambda prompts: enc(prompts)[0]
    else:
        enc = PromptEncoder("t5", max_length=24, dtype=torch.float32, configs=[t5_config(2, 32, 4, 64, 300)], native_attention=True)
        enc.load_model()
        model, call = enc.encoders[0].model, lambda prompts: enc(prompts, with_attention_mask=True)[0]
    sets = [PROMPTS, PROMPTS[::-1]]
    want = [call(p) for p in sets]
    both, got, errors = threading.Barrier(2, timeout=60), [None, None], []
    first = model.layers[0] if kind == "llama" else model.encoder.block[0]

    def wait(*_):           # neither begins ahead of the other's preparation
        both.wait()

    hook = first.register_forward_pre_hook(wait)

    def work(i):
        try:
            got[i] = call(sets[i])
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    hook.remove()
    assert not errors
    # the same sums in the same order, but for the products' own threads
    assert all(torch.allclose(a, b, atol=1e-5, rtol=0) for a, b in zip(want, got)) and not torch.allclose(want[0], want[1], atol=1e-2)


def test_a_model_that_was_not_prepared_says_so():
    import threading
    enc = _llama(native_attention=True)[1]
    ids = torch.ones(1, 5, dtype=torch.long)
    with pytest.raises(ValueError, match="prepare"):
        enc.model(input_ids=ids, use_cache=False)
    enc.native.prepare(None, 1, 5, "cpu")
    want = enc.model(input_ids=ids, use_cache=False).last_hidden_state
    got = []
    t = threading.Thread(target=lambda: got.append(enc.model(input_ids=ids, use_cache=False).last_hidden_state))       # one has prepared: its call goes on here
    t.start(), t.join()
    assert torch.allclose(got[0], want, atol=1e-5, rtol=0)
    import pickle
    copied = copy.deepcopy(enc)
    assert torch.equal(copied(PROMPTS)[0], enc(PROMPTS)[0])
    with pytest.raises(ValueError, match="prepare"):
        pickle.loads(pickle.dumps(enc.model))(input_ids=ids, use_cache=False)


@pytest.mark.gpu
def test_models_that_move_to_the_device_after_the_exchange():
    torch.manual_seed(4)
    cfg = llama_config(2, 256, 4, 2, 512, 1000)
    llama = LlamaTextEncoder(max_length=64, dtype=torch.float32, config=cfg, native_attention=True)
    t5 = PromptEncoder("t5", max_length=64, dtype=torch.float32, configs=[t5_config(2, 64, 2, 64, 300)], native_attention=True)
    t5.load_model()
    want = llama(PROMPTS)[0], t5(PROMPTS, with_attention_mask=True)[0]
    llama.model.to("cuda"), t5.encoders[0].model.to("cuda")
    got = llama(PROMPTS)[0], t5(PROMPTS, with_attention_mask=True)[0]
    # fp32 in the library's products on either side, states of the order of 1
    assert all(g.is_cuda and torch.allclose(g.cpu(), w, atol=2e-3, rtol=0) for g, w in zip(got, want))
    llama.model.to("cpu")
    assert torch.allclose(llama(PROMPTS)[0], want[0], atol=2e-4, rtol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_llama_on_the_kernels(dtype):
    """Heads of 128, shared, padded prompts; nearer to the fp32 states than a fiftieth, as the library's own are."""
    torch.manual_seed(2)
    cfg = llama_config(2, 512, 4, 2, 1024, 1000)
    exact = LlamaTextEncoder(max_length=256, dtype=torch.float32, config=cfg, device="cuda")
    native = copy.deepcopy(exact)
    native.model.to(dtype)
    native.native = use_native_attention(native.model)
    from teletron_b200.ops import _lib
    want, mask = exact(PROMPTS)
    before = _lib.LAUNCHES
    got, _ = native(PROMPTS)
    assert _lib.LAUNCHES - before == 2 + 2 * 2          # the plan, then rotation and attention of each layer
    assert float((got.float() - want)[mask].norm() / want[mask].norm()) < 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_t5_on_the_kernels(dtype):
    torch.manual_seed(3)
    exact = PromptEncoder("t5", max_length=300, dtype=torch.float32, configs=[t5_config(2, 256, 4, 512, 300)], device="cuda")
    exact.load_model()
    native = copy.deepcopy(exact)
    native.encoders[0].model.to(dtype)
    native.encoders[0].native = use_native_attention(native.encoders[0].model)
    long = [" ".join(f"w{i}" for i in range(250)), "a b c"]
    want, masks = exact(long, with_attention_mask=True)
    got, _ = native(long, with_attention_mask=True)
    keep = masks.bool().to(want.device)
    assert float((got.float() - want)[keep].norm() / want[keep].norm()) < 0.02
