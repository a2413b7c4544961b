"""The attention ops under Hugging Face causal LMs: an attention implementation ("crispybits") and a cache.

``install_attention(model)`` (integration.py) makes the model attend through ``prompt_attention`` and
``kv4_attention``; ``PagedKV4Cache`` is the cache to give it as ``past_key_values``.  A prompt attends to its own keys
and values as they come and stores them in 4 bits; every later token attends to what is stored, its own included.
Without a ``PagedKV4Cache`` every call must hold whole sequences (``use_cache=False``).

The attention is causal and unpadded: a batch with padding, a mask of its own, a sliding window, dropout, capped scores,
sinks or position biases raises ValueError.  Sequences of one batch have one length.  Needs transformers (imported here, not by the package).
"""
from __future__ import annotations

import torch
from transformers import AttentionInterface
from transformers.cache_utils import Cache, CacheLayerMixin
from transformers.masking_utils import AttentionMaskInterface, causal_mask_function

from .attention import KV4Cache, kv4_append, kv4_attention, prompt_attention

NAME = "crispybits"
_LAYER = "_crispybits_kv4_layer"          # where a layer's update leaves itself on the keys and values it returns
# arguments by which models ask for more than causal softmax attention
_OTHER = ("softcap", "s_aux", "position_bias", "head_mask", "indices", "block_indices", "cu_seq_lens_q", "cu_seq_lens_k")


class KV4Layer(CacheLayerMixin):
    """One layer's pages within a ``PagedKV4Cache``."""

    def __init__(self, owner: "PagedKV4Cache", cache: KV4Cache):
        super().__init__()
        self.owner, self.cache, self.seen, self.batch = owner, cache, 0, 0      # tokens and sequences held
        self.is_initialized = True

    def lazy_initialization(self, key_states, value_states):
        pass

    def update(self, key_states, value_states, *args, **kwargs):
        b, heads, s, d = key_states.shape
        o = self.owner
        n = self.seen + s
        if b > o.sequences or n > o.tokens:
            raise ValueError(f"{b} sequences of {n} tokens do not fit a cache of {o.sequences} x {o.tokens}")
        if self.seen and b != self.batch:
            raise ValueError(f"the cache holds {self.batch} sequences, not {b}")
        k, v = (t.transpose(1, 2).reshape(b * s, heads, d) for t in (key_states, value_states))
        kv4_append(self.cache, k, v, o.block_table[:b], o.lengths(n)[:b], None if s == 1 else o.starts(b, s))
        self.seen, self.batch = n, b
        # Behind earlier tokens the keys and values only stand for the cached ones (a view of the new ones, as long as all of
        # them): what a model makes of them is no longer this layer's, and too long to be taken for the new tokens' own.
        out = (key_states, value_states) if n == s else tuple(t[:, :, :1].expand(-1, -1, n, -1) for t in (key_states, value_states))
        for t in out:
            setattr(t, _LAYER, self)
        return out

    def get_mask_sizes(self, query_length: int):
        return self.seen + query_length, 0

    def get_seq_length(self) -> int:
        return self.seen

    def get_max_length(self) -> int:
        return self.owner.tokens

    def reset(self):
        self.seen = 0

    def crop(self, tokens_to_remove: int):
        """-n drops the newest n tokens (rejected drafts); a positive number, the older form, is the length to keep."""
        n = int(tokens_to_remove)
        self.seen = min(self.seen, n) if n > 0 else max(self.seen + n, 0)

    def batch_select_indices(self, indices: torch.Tensor):
        """Sequence i becomes sequence indices[i]."""
        n = indices.numel()
        if n > self.owner.sequences:
            raise ValueError("more sequences than the cache has room for")
        p = self.cache.pages.view(self.owner.sequences, -1, *self.cache.pages.shape[1:])
        p[:n] = p.index_select(0, indices.to(p.device))
        self.batch = n

    reorder_cache = batch_select_indices

    def batch_repeat_interleave(self, repeats: int):
        raise NotImplementedError("give the prompt once per sequence instead")

    def offload(self):
        raise NotImplementedError("the 4-bit cache stays on its device")

    prefetch = offload


class PagedKV4Cache(Cache):
    """Keys and values of every layer in 4 bits, for up to ``max_batch_size`` sequences of up to ``max_cache_len``
    tokens: a ``past_key_values`` for a model with ``install_attention``."""

    def __init__(self, config, max_batch_size: int, max_cache_len: int, device="cuda", page_size: int = 64):
        config = config.get_text_config()
        heads = config.num_attention_heads
        head_dim = getattr(config, "head_dim", None) or config.hidden_size // heads
        kv_heads = getattr(config, "num_key_value_heads", None) or heads
        self.sequences, self.tokens = int(max_batch_size), int(max_cache_len)
        pages = -(-self.tokens // page_size)
        self.block_table = torch.arange(self.sequences * pages, dtype=torch.int32, device=device).view(-1, pages)
        self.seq_lens = torch.zeros(self.sequences, dtype=torch.int32, device=device)
        self._length = 0                   # what seq_lens holds
        self._starts = {}
        super().__init__(layers=[KV4Layer(self, KV4Cache.empty(self.sequences * pages, kv_heads, head_dim, page_size,
                                                               device)) for _ in range(config.num_hidden_layers)])

    def lengths(self, n: int) -> torch.Tensor:
        """seq_lens, at n: one fill a step, the layers of a step share it.  The count is the host's, so a captured step
        would replay at one length."""
        if self.seq_lens.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKV4Cache counts tokens on the host: a captured step calls kv4_append and kv4_attention "
                               "with lengths of its own")
        if self._length != n:
            self.seq_lens.fill_(n)
            self._length = n
        return self.seq_lens

    def starts(self, b: int, s: int) -> torch.Tensor:
        """cu_seqlens of b sequences of s rows (the last one asked for is kept)."""
        if (b, s) not in self._starts:
            self._starts = {(b, s): _starts(b, s, self.seq_lens.device)}
        return self._starts[b, s]


def _starts(b: int, s: int, device) -> torch.Tensor:
    return torch.arange(0, (b + 1) * s, s, dtype=torch.int32, device=device)


def _mask(batch_size=None, q_length=None, kv_length=None, mask_function=causal_mask_function, attention_mask=None, **kwargs):
    """No mask is made; what the ops cannot do is refused."""
    if mask_function is not causal_mask_function:
        raise ValueError("crispybits attention is plainly causal: no sliding window, packed positions or mask function")
    if attention_mask is not None and not bool(attention_mask.all()):
        raise ValueError("crispybits attention takes no padding: give it prompts of one length")
    return None


def _attend(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    if attention_mask is not None or dropout or not getattr(module, "is_causal", True):
        raise ValueError("crispybits attention is causal, without a mask of its own and without dropout")
    if kwargs.get("sliding_window") is not None:
        raise ValueError("crispybits attention has no sliding window")
    b, heads, s, d = query.shape
    other = [n for n in _OTHER if kwargs.get(n) is not None]
    if other or (s > 1 and kwargs.get("is_causal") is False):
        raise ValueError(f"crispybits attention is plainly causal softmax attention: no {', '.join(other) or 'is_causal=False'}")
    q = query.transpose(1, 2)
    layer = getattr(key, _LAYER, None)
    if layer is not None and layer.seen > s and getattr(value, _LAYER, None) is layer:
        o = layer.owner
        return kv4_attention(q, layer.cache, o.block_table[:b], o.lengths(layer.seen)[:b], scale=scaling), None
    if key.shape[2] != s:
        raise ValueError("crispybits attention over earlier tokens needs a PagedKV4Cache as past_key_values, and the keys and "
                         "values that its update returned unchanged")
    k, v = (t.transpose(1, 2).reshape(b * s, -1, d) for t in (key, value))
    cu = layer.owner.starts(b, s) if layer is not None else _starts(b, s, q.device)
    return prompt_attention(q.reshape(b * s, heads, d), k, v, cu, s, scale=scaling).view(b, s, heads, d), None


def register():
    """The implementation under its name (again is fine)."""
    AttentionInterface.register(NAME, _attend)
    AttentionMaskInterface.register(NAME, _mask)
