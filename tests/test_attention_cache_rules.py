"""``PagedKV4Cache`` under the rules that Hugging Face's caches follow, on the CPU oracle in float64: what a crop keeps,
generation with drafted tokens that are checked and dropped, and models that do more to keys or scores than the ops know."""
from types import SimpleNamespace

import pytest
import torch

transformers = pytest.importorskip("transformers")

from transformers.cache_utils import DynamicCache  # noqa: E402

from crispybits_kernels import install_attention, kv4_cache, ops  # noqa: E402
from oracle import attention as O  # noqa: E402
from oracle import emulator  # noqa: E402


@pytest.fixture(autouse=True)
def cpu():
    prev = ops._C
    both = {n: getattr(emulator, n) for n in dir(emulator) if not n.startswith("_")}
    both.update({n: getattr(O, n) for n in ("kv4_page_words", "kv4_append", "kv4_read", "kv4_attention", "prompt_attention")})
    ops.set_backend(SimpleNamespace(**both))
    yield
    ops.set_backend(prev)


def _llama(**kw):
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(**{**dict(hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                                             num_key_value_heads=2, vocab_size=128), **kw})
    return install_attention(transformers.LlamaForCausalLM(cfg).double().eval())


def test_crop_keeps_what_a_dynamic_cache_keeps():
    """A negative number removes that many tokens, a positive one (the older form) is the length to keep."""
    model = _llama()
    tokens = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(1))
    for crops in ([-3], [-9], [-20], [0], [4], [9], [30], [-2, 5, -1]):
        cache, plain = kv4_cache(model, 2, 32, 32), DynamicCache()
        plain.update(torch.zeros(2, 2, 9, 16), torch.zeros(2, 2, 9, 16), 0)
        with torch.no_grad():
            model(tokens, past_key_values=cache)
            for n in crops:
                cache.crop(n)
                plain.crop(n)
            assert cache.get_seq_length() == plain.get_seq_length(), crops
            kept = cache.get_seq_length()
            if kept < 9:                                       # the removed tokens, fed again, are the newest ones
                again = model(tokens[:, kept:], past_key_values=cache).logits
                assert cache.get_seq_length() == 9
                whole = kv4_cache(model, 2, 32, 32)
                want = [model(t, past_key_values=whole).logits for t in (tokens[:, :kept], tokens[:, kept:]) if t.shape[1]]
                torch.testing.assert_close(again, want[-1], atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("drafts", [dict(prompt_lookup_num_tokens=4), dict(assistant=True)])
def test_checked_drafts_give_the_greedy_tokens(drafts):
    """Drafted tokens that are not accepted leave the cache: the tokens and the number cached are those of greedy decoding."""
    model = _llama()
    g = torch.Generator().manual_seed(2)
    part = torch.randint(0, 128, (1, 4), generator=g)
    prompt = torch.cat([part, torch.randint(0, 128, (1, 5), generator=g), part], 1)
    if drafts.pop("assistant", None):
        torch.manual_seed(3)
        drafts["assistant_model"] = transformers.LlamaForCausalLM(transformers.LlamaConfig(
            hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=2, vocab_size=128)).eval()
    got, lengths = [], []
    for kw in ({}, drafts):
        cache = kv4_cache(model, 1, 64, 32)
        got.append(model.generate(prompt, attention_mask=torch.ones_like(prompt), past_key_values=cache, max_new_tokens=12,
                                  do_sample=False, eos_token_id=None, pad_token_id=0, **kw))
        lengths.append(cache.get_seq_length())
    assert torch.equal(got[0], got[1])
    assert lengths == [24, 24]


def test_keys_changed_behind_the_update_are_refused():
    """JetMoe repeats keys and values after the cache took them: a prompt attends to them as they are, a later token, for
    which they stand for the cached ones, is refused rather than attending to itself alone."""
    torch.manual_seed(0)
    cfg = transformers.JetMoeConfig(hidden_size=64, intermediate_size=64, num_hidden_layers=2, num_key_value_heads=2, kv_channels=16,
                                    num_local_experts=4, num_experts_per_tok=2, vocab_size=128)
    plain = transformers.JetMoeForCausalLM(cfg).eval()
    tokens = torch.randint(0, 128, (1, 9), generator=torch.Generator().manual_seed(4))
    with torch.no_grad():
        want = plain(tokens).logits
        model = install_attention(plain)
        cache = kv4_cache(model, 1, 32, 32)
        torch.testing.assert_close(model(tokens, past_key_values=cache).logits, want, atol=1e-4, rtol=1e-4)
        with pytest.raises(ValueError, match="needs a PagedKV4Cache.*unchanged"):
            model(tokens[:, :1], past_key_values=cache)


@pytest.mark.parametrize("what", ["key", "value"])
def test_a_copy_of_what_the_update_returned_is_refused(what):
    from crispybits_kernels import hf_attention as H
    model = _llama()
    cache = kv4_cache(model, 1, 32, 32)
    g = torch.Generator().manual_seed(5)
    new = lambda n: [torch.randn(1, 2, n, 16, generator=g).double() for _ in range(2)]     # noqa: E731
    module = SimpleNamespace(is_causal=True)
    q = torch.randn(1, 4, 5, 16, generator=g).double()
    k, v = cache.update(*new(5), 0)
    first = H._attend(module, q, k, v, None)[0]
    assert torch.equal(H._attend(module, q, k.clone(), v.clone(), None)[0], first)           # a prompt holds all it needs
    k, v = cache.update(*new(1), 0)
    assert k.shape == v.shape == (1, 2, 6, 16)                                               # as a cache's keys and values are
    assert H._attend(module, q[:, :, :1], k, v, None)[0].shape == (1, 1, 4, 16)
    k, v = (t.clone() if what == n else t for n, t in (("key", k), ("value", v)))
    with pytest.raises(ValueError, match="needs a PagedKV4Cache.*unchanged"):
        H._attend(module, q[:, :, :1], k, v, None)


@pytest.mark.parametrize("kw", [dict(softcap=30.0), dict(s_aux=torch.zeros(4)), dict(sliding_window=8), dict(is_causal=False),
                                dict(position_bias=torch.zeros(1, 4, 5, 5)), dict(indices=torch.zeros(1, 5, 2)),
                                dict(cu_seq_lens_q=torch.tensor([0, 2, 5]))])
def test_other_attentions_are_refused(kw):
    """Arguments that would change the result are not dropped."""
    from crispybits_kernels import hf_attention as H
    q = torch.zeros(1, 4, 5, 16)
    module = SimpleNamespace(is_causal=True)
    with pytest.raises(ValueError, match="crispybits attention"):
        H._attend(module, q, q, q, None, **kw)
    H._attend(module, q, q, q, None, **{k: None for k in kw}, position_ids=torch.arange(5)[None], use_cache=True)


def test_a_batch_keeps_its_size():
    """A later token of more or fewer sequences than the cached ones is refused; choosing sequences changes their number."""
    model = _llama()
    tokens = torch.randint(0, 128, (3, 5), generator=torch.Generator().manual_seed(6))
    with torch.no_grad():
        cache = kv4_cache(model, 3, 32, 32)
        model(tokens[:2], past_key_values=cache)
        for b in (1, 3):
            with pytest.raises(ValueError, match="holds 2 sequences"):
                model(tokens[:b, :1], past_key_values=cache)
        assert cache.get_seq_length() == 5
        cache.batch_select_indices(torch.tensor([1]))
        got = model(tokens[1:2, :1], past_key_values=cache).logits
        one = kv4_cache(model, 1, 32, 32)
        model(tokens[1:2], past_key_values=one)
        torch.testing.assert_close(got, model(tokens[1:2, :1], past_key_values=one).logits, atol=1e-5, rtol=1e-5)
        cache.reset()
        model(tokens, past_key_values=cache)
        assert cache.get_seq_length() == 5
