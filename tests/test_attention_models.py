"""The attention ops under whole models: tiny Llama and OPT LMs with ``install_attention`` and a ``PagedKV4Cache``
against the same models attending in plain torch over a cache that holds what the 4-bit cache holds.

On the CPU oracle in float32 (host logic: layouts, lengths, refusals), and on the GPU with packed linears through
``install_bitmap(attention=True)``."""
import copy
from types import SimpleNamespace

import pytest
import torch

transformers = pytest.importorskip("transformers")

from transformers.cache_utils import Cache, DynamicLayer  # noqa: E402

from crispybits_kernels import install_attention, install_bitmap, kv4_cache, ops  # noqa: E402
from crispybits_kernels.reference import write_packed_dir  # noqa: E402
from oracle import attention as O  # noqa: E402
from oracle import emulator  # noqa: E402


class _Held(DynamicLayer):
    """A layer that gives a prompt its own keys and values and later tokens what 4 bits hold of everything."""

    def update(self, key_states, value_states, *args, **kwargs):
        first = self.get_seq_length() == 0
        held = [torch.from_numpy(O.values(*O.quantize(t.detach().cpu().double().numpy()))).to(t) for t in (key_states, value_states)]
        k, v = super().update(*held)
        return (key_states, value_states) if first else (k, v)


def _model(kind, heads=4, kv=2, hidden=160):
    torch.manual_seed(0)
    if kind == "llama":
        cfg = transformers.LlamaConfig(hidden_size=hidden, intermediate_size=256, num_hidden_layers=2, num_attention_heads=heads,
                                       num_key_value_heads=kv, vocab_size=128)
        m = transformers.LlamaForCausalLM(cfg)
        with torch.no_grad():
            for blk in m.model.layers:
                blk.self_attn.q_proj.weight.mul_(8.0)
                blk.self_attn.k_proj.weight.mul_(8.0)
    else:
        cfg = transformers.OPTConfig(hidden_size=hidden, ffn_dim=256, num_hidden_layers=2, num_attention_heads=heads,
                                     vocab_size=128, word_embed_proj_dim=hidden)
        m = transformers.OPTForCausalLM(cfg)
    return m.eval()


@pytest.fixture
def cpu():
    prev = ops._C
    both = {n: getattr(emulator, n) for n in dir(emulator) if not n.startswith("_")}
    both.update({n: getattr(O, n) for n in ("kv4_page_words", "kv4_append", "kv4_read", "kv4_attention", "prompt_attention")})
    ops.set_backend(SimpleNamespace(**both))
    yield
    ops.set_backend(prev)


def _steps(model, cache, tokens, chunks):
    """Logits of the chunks fed one after another."""
    out, at = [], 0
    with torch.no_grad():
        for n in chunks:
            out.append(model(tokens[:, at:at + n], past_key_values=cache, use_cache=True).logits)
            at += n
    return torch.cat(out, 1)


@pytest.mark.parametrize("kind", ["llama", "opt"])
def test_model_on_the_oracle(cpu, kind):
    """A prompt, single tokens, a chunk of three, a crop, more tokens; two sequences; pages of 32 crossed."""
    plain = _model(kind)
    model = install_attention(copy.deepcopy(plain))
    plain.set_attn_implementation("eager")
    tokens = torch.randint(0, 128, (2, 45), generator=torch.Generator().manual_seed(1))
    chunks = [29, 1, 1, 3, 1]
    cache = kv4_cache(model, 3, 64, 32)
    want_cache = Cache(layer_class_to_replicate=_Held)
    got, want = _steps(model, cache, tokens, chunks), _steps(plain, want_cache, tokens, chunks)
    torch.testing.assert_close(got, want, atol=2e-4, rtol=2e-4)
    assert cache.get_seq_length() == 35 and cache.get_max_length() == 64
    cache.crop(2)
    for layer in want_cache.layers:
        layer.keys, layer.values = layer.keys[:, :, :-2], layer.values[:, :, :-2]
    got, want = _steps(model, cache, tokens[:, 33:], [1, 2]), _steps(plain, want_cache, tokens[:, 33:], [1, 2])
    torch.testing.assert_close(got, want, atol=2e-4, rtol=2e-4)
    swap = torch.tensor([1, 0])
    cache.reorder_cache(swap)
    want_cache.reorder_cache(swap)
    t = tokens.flip(0)
    torch.testing.assert_close(_steps(model, cache, t[:, 36:], [1]), _steps(plain, want_cache, t[:, 36:], [1]), atol=2e-4, rtol=2e-4)


def test_model_without_a_cache(cpu):
    plain = _model("llama")
    model = install_attention(copy.deepcopy(plain))
    tokens = torch.randint(0, 128, (2, 20), generator=torch.Generator().manual_seed(2))
    with torch.no_grad():
        torch.testing.assert_close(model(tokens, use_cache=False).logits, plain(tokens, use_cache=False).logits, atol=2e-4, rtol=2e-4)


def test_model_refusals(cpu):
    model = install_attention(_model("llama"))
    tokens = torch.zeros(2, 6, dtype=torch.long)
    pad = torch.ones(2, 6, dtype=torch.long)
    with torch.no_grad():
        model(tokens, attention_mask=pad, past_key_values=kv4_cache(model, 2, 32, 32))
        pad[0, :2] = 0
        with pytest.raises(ValueError, match="no padding"):
            model(tokens, attention_mask=pad, past_key_values=kv4_cache(model, 2, 32, 32))
        with pytest.raises(ValueError, match="do not fit"):
            model(tokens, past_key_values=kv4_cache(model, 1, 32, 32))
        cache = kv4_cache(model, 2, 8, 32)
        model(tokens, past_key_values=cache)
        with pytest.raises(ValueError, match="do not fit"):
            model(tokens[:, :3], past_key_values=cache)
        with pytest.raises(ValueError, match="mask of its own"):
            model(tokens, attention_mask=torch.zeros(2, 1, 6, 6), use_cache=False)
        out = model(tokens, use_cache=True)                      # the model makes a cache of its own
        with pytest.raises(ValueError, match="needs a PagedKV4Cache"):
            model(tokens[:, :1], past_key_values=out.past_key_values)


def test_masks_and_refused_updates_of_later_steps(cpu):
    """A mask that hides an earlier token is refused at single tokens too; a refused update and a crop by less than
    nothing leave the count of tokens as it was."""
    model = install_attention(_model("llama"))
    tokens = torch.zeros(2, 6, dtype=torch.long)
    cache = kv4_cache(model, 2, 8, 32)
    with torch.no_grad():
        model(tokens, past_key_values=cache)
        mask = torch.ones(2, 7, dtype=torch.long)
        mask[1, 0] = 0
        with pytest.raises(ValueError, match="no padding"):
            model(tokens[:, :1], attention_mask=mask, past_key_values=cache)
        with pytest.raises(ValueError, match="do not fit"):
            model(tokens[:, :3], past_key_values=cache)
        cache.crop(-3)
        assert cache.get_seq_length() == 6
        model(tokens[:, :1], attention_mask=torch.ones(2, 7, dtype=torch.long), past_key_values=cache)
        assert cache.get_seq_length() == 7


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,hidden", [("llama", 4, 2, 256), ("llama", 4, 4, 512), ("opt", 4, 4, 320)])
def test_packed_model(hip, tmp_path, monkeypatch, kind, heads, kv, hidden):
    """Packed linears and 4-bit cache together, prompt then decode steps (fused RoPE on Llama).  Each attention call is
    held to float64 attention over its own inputs and what its layer's cache holds at that moment: whole logits of two
    such models part where a rounding upstream moves a code by a step.  A prompt's output is rounded once and its
    weights once (2^-10 of sum p |v| together, twice that allowed); over the cache the codes are exact, the weights rounded
    once, and codes and zero points summed apart in fp32: for n <= 64 tokens n / 4 + 16 <= 32 roundings, each half a last
    place (2^-24) of at most 30 s <= 4 max |v| (s <= 2 max |v| / 15), less than 2^-16 max |v| in all."""
    from crispybits_kernels import hf_attention as H
    base = _model(kind, heads, kv, hidden).half().cuda()
    bitmap = [4, 3]
    write_packed_dir(copy.deepcopy(base).cpu(), tmp_path, bitmap=bitmap)
    calls = []
    real = H._attend

    def checked(module, query, key, value, *args, **kwargs):
        out, _ = real(module, query, key, value, *args, **kwargs)
        b, _, n, d = query.shape
        scale = kwargs.get("scaling") or d ** -0.5
        q, k, v = (t.transpose(1, 2).reshape(b * n, -1, d) for t in (query, key, value))
        layer = getattr(key, H._LAYER)
        if layer.seen == n:
            want, mag = O.prompt64(q, k, v, torch.arange(0, (b + 1) * n, n), scale)
        else:
            want, mag = O.attention64(q.view(b, n, -1, d), layer.cache.pages, layer.cache.page_size, d,
                                      layer.owner.block_table[:b], torch.full((b,), layer.seen), scale)
        err = abs(out.double().cpu().numpy().reshape(want.shape) - want)
        held = [O.stored(layer.cache.pages, layer.cache.page_size, d, layer.owner.block_table, i, layer.seen)[1]
                for i in range(b)]
        top = max(abs(t).max() for t in held)
        calls.append(float((err / (2.0 ** -9 * mag + 2.0 ** -16 * top + 1e-6)).max()))
        return out, None

    monkeypatch.setattr(H, "_attend", checked)
    model = install_bitmap(copy.deepcopy(base), str(tmp_path), bitmap, attention=True)
    tokens = torch.randint(0, 128, (2, 60), generator=torch.Generator().manual_seed(3)).cuda()
    chunks = [50, 1, 1, 4, 1, 1, 1]
    logits = _steps(model, kv4_cache(model, 2, 128, 32), tokens, chunks)
    assert torch.isfinite(logits).all()
    assert len(calls) == 2 * len(chunks) and max(calls) <= 1.0, calls
    ids = model.generate(tokens[:, :20], attention_mask=torch.ones_like(tokens[:, :20]), past_key_values=kv4_cache(model, 2, 64),
                         max_new_tokens=8, do_sample=False)
    assert ids.shape == (2, 28) and torch.equal(ids[:, :20], tokens[:, :20])
    monkeypatch.setattr(H, "_attend", real)
    H.register()
