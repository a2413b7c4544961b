"""Scores far from zero, of either sign, up to the edge of fp32: softmax of finite scores is finite.

Keys take few values and queries one, so that scores are exact products with ties, and different scores lie so far apart that
a row's softmax is even over the visible tokens of its largest score.  Bound of an output: its own rounding, the weights' (half a step
of the type; over the cache 2^-11, fp32 2^-22), 2^-20 for the exponentials and the fp32 sums; over the cache these are (n / 4 + 16)
roundings of at most 30 times the largest p s', and fp16 may lose 2^-31 of that for each token (test_gpu_kv4_peaks.py)."""
import numpy as np
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_attention, prompt_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
POWERS = [20, 23, 24, 25, 27, 31, 32, 40, 64, 100, 122, 125]


def _close(got, want, mag, dtype, n, vmax, weight=None):
    step = torch.finfo(dtype).eps / 2
    share = (step if weight is None else weight) + (n + 16) * 2.0 ** -24 + 2.0 ** -20
    tol = step * np.abs(want) + share * mag + n * 2.0 ** -28 * vmax
    diff = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert np.isfinite(diff).all() and (diff <= tol).all(), float(np.nanmax(diff / tol))


def _keys(n, heads, d, g):
    """Values of one of eight sizes at place 3: 1, 1 + 2^-6 .. 1 + 7 2^-6 in fp32 (exact in bf16)."""
    k = torch.zeros(n, heads, d)
    k[..., 3] = 1 + torch.randint(0, 8, (n, heads), generator=g) / 64
    return k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_prompts(hip, dtype, sign, d):
    lens = [150, 1, 70]
    g = torch.Generator().manual_seed(d)
    n = sum(lens)
    q, k, v = torch.zeros(n, 4, d), _keys(n, 2, d, g), torch.randn(n, 2, d, generator=g)
    q[..., 3] = sign
    q[:, 3, 3] = sign * 2.0 ** -30                                      # a head of ordinary scores beside it
    k[20, 0, 3] = 0.5                                                   # the largest, or the smallest, far down the sequence
    cu = torch.tensor([0, 150, 151, 221], dtype=torch.int32)
    q, k, v = (t.to(dtype) for t in (q, k, v))
    if dtype == torch.float16:
        q[:, 3, 3] = sign * 2.0 ** -14
    for p in POWERS:
        scale = 2.0 ** p
        got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 150, scale=scale)

        want, mag = O.prompt64(q, k, v, cu, scale)
        _close(got[:, :3], want[:, :3], mag[:, :3], dtype, 150, 4.0)
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompts_of_large_inputs(hip, dtype):
    """Products below -1e30 by the inputs' own size."""
    g = torch.Generator().manual_seed(9)
    q, k, v = torch.zeros(140, 2, 64), _keys(140, 2, 64, g), torch.randn(140, 2, 64, generator=g)
    for a, b in ((-2.0 ** 60, 2.0 ** 55), (2.0 ** 60, 2.0 ** 55), (-2.0 ** 110, 2.0 ** 5)):
        q[..., 3] = a
        qq, kk, vv = (t.to(dtype) for t in (q, k * b, v))
        cu = torch.tensor([0, 140], dtype=torch.int32)
        got = prompt_attention(qq.cuda(), kk.cuda(), vv.cuda(), cu.cuda())
        want, mag = O.prompt64(qq, kk, vv, cu, 64 ** -0.5)
        _close(got, want, mag, dtype, 140, 4.0)


def _cache(lens, k, v, page):
    table = torch.full((len(lens), max(-(-n // page) for n in lens)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        need = -(-n // page)
        table[b, :need] = torch.arange(at, at + need)
        at += need
    pages = torch.zeros(at, k.shape[1], O.kv4_page_words(k.shape[2], page), dtype=torch.int32)
    ln = torch.tensor(lens, dtype=torch.int32)
    O.kv4_append(pages, page, k.shape[2], k, v, table, ln, torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32))
    return pages, table, ln


def _cache_check(q, pages, page, table, ln, scale, heads):
    """q [sequences, t, heads, d] over the cache, `heads` of it within the bound."""
    dtype, d, t = q.dtype, q.shape[3], q.shape[1]
    group = q.shape[2] // pages.shape[1]
    got = kv4_attention(q.cuda(), KV4Cache(pages.cuda(), page, d), table.cuda(), ln.cuda(), scale=scale)
    assert torch.isfinite(got).all()
    got = got.double().cpu().numpy()
    words = pages.numpy().view(np.uint32).reshape(pages.shape[0], pages.shape[1], -1, O._block_words(d))
    step, weight = torch.finfo(dtype).eps / 2, 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    for b, n in enumerate(ln.tolist()):
        k, v, _ = O.stored(pages, page, d, table, b, n)
        at = 256 * -(-d // 32) + 32
        sv = np.array([words[int(table[b, i // page]), :, i % page // 32, at + i % 32] for i in range(n)], np.uint32).view(np.float32)
        for i in range(t):
            m = n - t + i + 1
            for h in heads:
                kh, vh = (a[:m, h // group].astype(np.float64) for a in (k, v))
                s = scale * (kh @ q[b, i, h].double().numpy())
                p = np.exp(s - s.max())
                p /= p.sum()
                top = (p * sv[:m, h // group].astype(np.float64)).max()
                want, mag = p @ vh, p @ np.abs(vh)
                tol = step * np.abs(want) + (weight + 2.0 ** -20) * mag + ((m / 4 + 16) * 2.0 ** -24 * 30 + m * 2.0 ** -31 * 15) * top
                diff = np.abs(got[b, i, h] - want)
                assert (diff <= tol).all(), (b, i, h, float((diff / tol).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_cached(hip, dtype, sign):
    """Short and long sequences (several workgroups to one), two new tokens each; a head of ordinary scores beside the far ones."""
    lens, d, page = [150, 2, 70, 2500], 64, 64
    g = torch.Generator().manual_seed(11)
    n = sum(lens)
    k, v = _keys(n, 2, d, g), torch.randn(n, 2, d, generator=g) * torch.exp2(torch.randint(-3, 4, (n, 2, 1), generator=g).float())
    k[20, 0, 3], k[60, 1, 3] = 0.5, 2.0
    pages, table, ln = _cache(lens, k, v, page)
    q = torch.zeros(4, 2, 4, d)
    q[..., 3] = sign
    q[:, :, 3, 3] = sign * 2.0 ** -14
    q = q.to(dtype)
    for p in POWERS:
        _cache_check(q, pages, page, table, ln, 2.0 ** p, [0, 1, 2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_cached_large_inputs(hip, dtype):
    """Queries and keys of large and small sizes whose scores are far from zero, values of any scale: the largest score's tokens count
    whatever their values' scale beside the others'."""
    lens, d, page = [150, 333], 64, 32
    g = torch.Generator().manual_seed(12)
    n = sum(lens)
    for a, b, scale in ((-2.0 ** 60, 2.0 ** 55, 0.125), (2.0 ** 60, 2.0 ** 55, 0.125), (-2.0 ** 120, 2.0 ** -20, 0.5),
                        (2.0 ** 125, 2.0 ** -40, 4.0), (2.0 ** -100, 2.0 ** 30, 2.0 ** 110)):
        for vp in (0, 90, -60):
            k = _keys(n, 1, d, g) * b
            tie = (k[..., 3] == k[..., 3].max()) if a > 0 else (k[..., 3] == k[..., 3].min())
            v = torch.randn(n, 1, d, generator=g) * 2.0 ** vp
            v = torch.where(tie[..., None], v, v * 2.0 ** 30)              # what has no weight is large
            pages, table, ln = _cache(lens, k, v, page)
            q = torch.zeros(2, 1, 2, d)
            q[..., 3] = a
            _cache_check(q.to(dtype), pages, page, table, ln, scale, [0, 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,scale", [(2.0 ** -130, 2.0 ** -30), (2.0 ** -24, 2.0 ** -140), (0.0, 2.0 ** -149), (2.0 ** -133, 2.0 ** -149)])
def test_cached_scores_of_nothing(hip, dtype, size, scale):
    """Queries and scales whose factor is below the smallest float: an even softmax, with hidden tokens in every block."""
    lens, d, page = [1, 20, 45], 64, 32
    g = torch.Generator().manual_seed(13)
    n = sum(lens)
    k, v = torch.randn(n, 1, d, generator=g), torch.randn(n, 1, d, generator=g)
    pages, table, ln = _cache(lens, k, v, page)
    q = (torch.randn(3, 1, 2, d, generator=g).sign().double() * size).to(dtype)
    _cache_check(q, pages, page, table, ln, scale, [0, 1])
