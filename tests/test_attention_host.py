"""The attention entry points without a GPU: the C ABI of include/crispybits_attention.h (exports, argument
checks before any HIP call, empty calls), the package's host logic on the CPU oracle, and the oracle's cache format."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import crispybits_kernels as ck
from crispybits_kernels import _C, ops
from oracle import attention as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "crispybits_attention.h")
P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
SIGS = {
    "cbk_kv4_page_words": (L, [I, L]),
    "cbk_kv4_append": (I, [P, L, L, I, L, P, P, I, L, L, L, L, L, P, L, P, P, L, I, P]),
    "cbk_kv4_read": (I, [P, L, L, I, L, P, P, I, L, P, L, P, P, L, I, P]),
    "cbk_kv4_attention_partial_floats": (L, [L, L, L, L, I, L, L]),
    "cbk_kv4_attention": (I, [P, I, L, L, L, P, L, L, I, L, P, L, P, F, P, L, P, I, P]),
    "cbk_prompt_attention": (I, [P, P, P, I, L, L, L, I, L, L, L, L, L, L, P, L, L, F, I, P, I, P]),
}
lib = ctypes.CDLL(_C.LIB_PATH)
for _n, (_r, _a) in SIGS.items():
    getattr(lib, _n).restype, getattr(lib, _n).argtypes = _r, _a
lib.cbk_last_error.restype = ctypes.c_char_p
ALIGNED = 1 << 20          # a fake, 16-byte aligned "device" address: never dereferenced


def _err():
    return lib.cbk_last_error().decode()


def test_header_and_library_agree():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    assert set(re.findall(r"\b(cbk_\w+)\s*\(", text)) == set(SIGS)
    for name in SIGS:
        assert hasattr(lib, name)


def test_page_words():
    assert lib.cbk_kv4_page_words(128, 64) == 2 * 1088
    assert lib.cbk_kv4_page_words(80, 32) == 832
    for d, page in ((128, 48), (128, 16), (128, 0), (128, 131072), (12, 32), (0, 32), (264, 32), (-8, 32)):
        assert lib.cbk_kv4_page_words(d, page) == -1
        with pytest.raises(RuntimeError, match="head_dim must be"):
            _C.kv4_page_words(d, page)
    for d in (8, 64, 80, 200, 256):
        assert lib.cbk_kv4_page_words(d, 64) == O.kv4_page_words(d, 64)


def _append(**kw):
    a = dict(pages=ALIGNED, num_pages=4, heads=2, d=128, page=64, k=ALIGNED, v=ALIGNED, dtype=0, rows=3, kr=256, kh=128,
             vr=256, vh=128, table=ALIGNED, width=2, lens=ALIGNED, cu=ALIGNED, seqs=2, device=0, stream=None)
    a.update(kw)
    return lib.cbk_kv4_append(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "fp16/bf16/fp32"), (dict(d=12), "head_dim must be"), (dict(d=264), "head_dim must be"),
    (dict(heads=0), "heads must be"), (dict(page=48), "page_size must be"), (dict(num_pages=-1), "number of pages"),
    (dict(kr=252), "16-byte aligned"), (dict(vh=4), "16-byte aligned"), (dict(dtype=2, vh=6), "16-byte aligned"),
    (dict(kr=-256), "16-byte aligned"), (dict(k=ALIGNED + 8), "16-byte aligned"), (dict(pages=ALIGNED + 4), "16-byte aligned"),
    (dict(table=None), "non-null"), (dict(lens=None), "non-null"), (dict(pages=None), "non-null"), (dict(v=None), "non-null"),
    (dict(cu=None), "one row a sequence"), (dict(rows=-1), "number of rows"), (dict(seqs=70000), "at most"),
    (dict(width=1 << 30), "too wide"), (dict(rows=(1 << 28) + 1), "number of rows"),
])
def test_append_refusals(kw, msg):
    assert _append(**kw) == 1 and msg in _err()


def test_empty_calls_are_no_ops():
    assert _append(rows=0) == 0
    assert _append(rows=0, seqs=0, cu=None) == 0
    assert _read(rows=0) == 0
    assert _attention(seqs=0) == 0
    assert _attention(t=0) == 0
    assert _prompt(rows=0, longest=0) == 0


def _read(**kw):
    a = dict(pages=ALIGNED, num_pages=4, heads=2, d=128, page=64, k=ALIGNED, v=ALIGNED, dtype=0, rows=3, table=ALIGNED,
             width=2, lens=ALIGNED, cu=ALIGNED, seqs=2, device=0, stream=None)
    a.update(kw)
    return lib.cbk_kv4_read(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=-1), "fp16/bf16/fp32"), (dict(page=33), "page_size must be"), (dict(k=ALIGNED + 2), "16-byte aligned"),
    (dict(k=None), "non-null"), (dict(cu=None), "one row a sequence"), (dict(seqs=0), "rows without a sequence"),
    (dict(rows=(1 << 28) + 1), "number of rows"),
])
def test_read_refusals(kw, msg):
    assert _read(**kw) == 1 and msg in _err()


def _attention(**kw):
    a = dict(q=ALIGNED, dtype=0, seqs=2, t=1, heads=4, pages=ALIGNED, num_pages=4, kv=2, d=128, page=64, table=ALIGNED,
             width=2, lens=ALIGNED, scale=0.1, partial=ALIGNED, floats=1 << 40, out=ALIGNED, device=0, stream=None)
    a.update(kw)
    return lib.cbk_kv4_attention(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=9), "fp16/bf16/fp32"), (dict(heads=3), "multiple of kv_heads"), (dict(kv=0), "multiple of kv_heads"),
    (dict(d=4), "head_dim must be"), (dict(scale=0.0), "scale must be"), (dict(scale=-1.0), "scale must be"),
    (dict(scale=float("nan")), "scale must be"), (dict(scale=float("inf")), "scale must be"), (dict(t=-1), "new tokens"),
    (dict(t=1 << 22), "too many new tokens"), (dict(q=None), "non-null"), (dict(out=ALIGNED + 4), "16-byte aligned"),
    (dict(seqs=60000, width=100000), "block table too wide"), (dict(floats=0, width=64), "partial must hold"), (dict(partial=None, width=64), "partial must hold"),
    (dict(lens=None), "non-null"), (dict(page=100), "page_size must be"),
])
def test_attention_refusals(kw, msg):
    assert _attention(**kw) == 1 and msg in _err()


def test_partial_floats():
    n = lib.cbk_kv4_attention_partial_floats
    assert n(1, 1, 32, 8, 128, 64, 1) == 0                      # units of two blocks are never cut
    for seqs, width in ((1, 64), (64, 64), (1, 2048)):          # two slots a workgroup of rows of sums and two more
        got = n(seqs, 1, 32, 8, 128, 64, width)
        assert got > 0 and got % (2 * 4 * 130) == 0
    for bad in ((0, 1, 32, 8, 128, 64, 64), (1, 1, 3, 2, 128, 64, 64), (1, 1, 2, 2, 12, 64, 64), (1, 1, 2, 2, 128, 48, 64)):
        assert n(*bad) == 0


def _prompt(**kw):
    a = dict(q=ALIGNED, k=ALIGNED, v=ALIGNED, dtype=0, rows=100, heads=4, kv=2, d=128, qr=512, qh=128, kr=256, kh=128, vr=256,
             vh=128, cu=ALIGNED, seqs=2, longest=80, scale=0.1, zero=1, out=ALIGNED, device=0, stream=None)
    a.update(kw)
    return lib.cbk_prompt_attention(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=4), "fp16/bf16/fp32"), (dict(heads=5), "multiple of kv_heads"), (dict(d=100), "head_dim must be"),
    (dict(qr=510), "16-byte aligned"), (dict(kr=1 << 24), "at most 2^23"), (dict(kh=4), "16-byte aligned"), (dict(vr=-8), "16-byte aligned"),
    (dict(v=ALIGNED + 8), "16-byte aligned"), (dict(cu=None), "non-null"), (dict(out=None), "non-null"),
    (dict(scale=0.0), "scale must be"), (dict(longest=0), "max_seqlen must be"), (dict(longest=101), "max_seqlen must be"),
    (dict(seqs=0), "rows without a sequence"), (dict(seqs=70000), "at most"), (dict(rows=-5), "number of rows"),
    (dict(rows=1 << 29, longest=1 << 29, heads=4, seqs=1000), "too large"),
    (dict(rows=1 << 22, longest=1 << 22, heads=4, seqs=128), "too large"),      # 2^15 x 129 x 4 workgroups of 256
])
def test_prompt_refusals(kw, msg):
    assert _prompt(**kw) == 1 and msg in _err()


def test_ops_refuse_cpu_tensors_and_wrong_ranks():
    x = torch.zeros(3, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q must be CUDA"):
        ck.prompt_attention(x, x, x, i)
    with pytest.raises(RuntimeError, match="k must be CUDA"):
        ck.kv4_append(ck.KV4Cache(torch.zeros(1, 2, 576, dtype=torch.int32), 32, 64), x, x, i[None], i)
    with pytest.raises(ValueError, match="q must be"):
        ck.prompt_attention(x[0], x, x, i)
    with pytest.raises(ValueError, match="q must be"):
        ck.kv4_attention(x[0], ck.KV4Cache(i, 32, 64), i, i)
    with pytest.raises(ValueError, match="number of packed rows"):
        ck.kv4_read(ck.KV4Cache(i, 32, 64), i, i, i)


def test_missing_library_is_reported(monkeypatch):
    monkeypatch.setattr(ops, "_C", None)
    with pytest.raises(RuntimeError, match="not built"):
        ck.KV4Cache.empty(1, 1, 64, 32, "cpu")


@pytest.fixture
def cpu_attention():
    prev = ops._C
    ops.set_backend(O)
    yield
    ops._C = prev


def test_serving_loop_on_the_oracle(cpu_attention):
    """Prompts, then decode steps, through the package on the oracle: the cache's attention equals attention over what
    the cache gives back, and defaults (scale, max_seqlen, one row a sequence) are passed through."""
    g = torch.Generator().manual_seed(0)
    d, hq, hkv, lens = 40, 4, 2, [5, 33]
    cache = ck.KV4Cache.empty(5, hkv, d, 32, "cpu")
    assert cache.num_pages == 5 and cache.num_kv_heads == 2
    table = torch.tensor([[4, -1], [1, 3]], dtype=torch.int32)
    cu = torch.tensor([0, 5, 38], dtype=torch.int32)
    q, k, v = (torch.randn(38, h, d, generator=g) for h in (hq, hkv, hkv))
    n = torch.tensor(lens, dtype=torch.int32)
    ck.kv4_append(cache, k, v, table, n, cu)
    o = ck.prompt_attention(q, k, v, cu)
    s = torch.nn.functional.scaled_dot_product_attention(
        q[5:].transpose(0, 1), k[5:].transpose(0, 1).repeat_interleave(2, 0), v[5:].transpose(0, 1).repeat_interleave(2, 0),
        is_causal=True).transpose(0, 1)
    torch.testing.assert_close(o[5:], s, atol=1e-5, rtol=1e-5)
    for _ in range(3):
        n += 1
        q1, k1, v1 = (torch.randn(2, h, d, generator=g) for h in (hq, hkv, hkv))
        ck.kv4_append(cache, k1, v1, table, n)
        got = ck.kv4_attention(q1, cache, table, n)
        cu_all = torch.tensor([0, int(n[0]), int(n.sum())], dtype=torch.int32)
        kk, vv = ck.kv4_read(cache, table, n, cu_all, int(n.sum()), torch.float32)
        for b in range(2):
            a, z = int(cu_all[b]), int(cu_all[b + 1])
            w = torch.nn.functional.scaled_dot_product_attention(
                q1[b][:, None], kk[a:z].transpose(0, 1).repeat_interleave(2, 0),
                vv[a:z].transpose(0, 1).repeat_interleave(2, 0))[:, 0]
            torch.testing.assert_close(got[b], w, atol=1e-5, rtol=1e-5)
        last = torch.stack([kk[int(cu_all[b + 1]) - 1] for b in range(2)])
        assert (last - k1).abs().max() <= 0.55 * (k1.amax(-1).clamp_min(0) - k1.amin(-1).clamp_max(0)).max() / 15


def test_oracle_places_are_a_permutation():
    """Every code of a block has a place of its own within the block's code words."""
    for d in (8, 80, 128, 200):
        ns = -(-d // 32)
        seen = set()
        for place, base in ((O.k_place, 0), (O.v_place, 128 * ns)):
            for t in range(32):
                for i in range(32 * ns):
                    x, bit = place(d, t, i)
                    assert base <= x < base + 128 * ns and bit % 4 == 2
                    seen.add((x, bit))
        assert len(seen) == 2 * 32 * 32 * ns


def test_oracle_quantizer():
    """Codes and words of chosen vectors."""
    x = np.array([[0.0] * 8, [-7.5, 7.5, 0, 0, 0, 0, 0, 0], [15.0, 1, 2, 3, 4.5, 5.5, 0, 0.25], [-15, -1, 0, 0, 0, 0, 0, 0],
                  [np.inf, 1, 1, 1, 1, 1, 1, 1]])
    c, w = O.quantize(x)
    v = O.values(c, w)
    assert not v[0].any()
    assert (w[1] & 15) == 8 and (w[2] & 15) == 0 and (w[3] & 15) == 15
    np.testing.assert_allclose(v[1, :2], [-7, 7], atol=1.01)
    assert list(c[2]) == [15, 1, 2, 3, 4, 6, 0, 0]
    np.testing.assert_allclose(v[3, :2], [-15, -1], rtol=1e-5)
    assert np.isnan(v[4]).all()
