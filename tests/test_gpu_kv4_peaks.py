"""Attention over the 4-bit cache where one token has nearly all of the probability and a tiny value vector, beside tokens
of huge value vectors and no probability.

Bound of an output: as in test_gpu_kv4.py its own rounding, each weight's (2^-11, fp32 2^-22) and twice the error of scores as shares of sum
p |v|; the fp32 sums over tokens, codes and zero points apart, (n / 4 + 16) roundings of at most 30 times the largest p s'; and what
fp16 loses of the smallest weights: the largest weight stands at 2^10 at least, half the smallest step is 2^-25, and counts up to
16-fold: 2^-31 of the largest p s' times at most 15 for each token."""
import numpy as np
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu


def _pages(lens, k, v, page):
    hkv, d = k.shape[1:]
    need = [-(-n // page) for n in lens]
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    pages = torch.zeros(at, hkv, O.kv4_page_words(d, page), dtype=torch.int32)
    ln = torch.tensor(lens, dtype=torch.int32)
    O.kv4_append(pages, page, d, k, v, table, ln, torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32))
    return pages, table, ln


def _scales(pages, d, table, page, b, n, h, value):
    words = pages.numpy().view(np.uint32).reshape(pages.shape[0], pages.shape[1], -1, O._block_words(d))
    at = 256 * -(-d // 32) + (32 if value else 0)
    return np.array([words[int(table[b, i // page]), h, i % page // 32, at + i % 32] for i in range(n)], np.uint32).view(np.float32).astype(np.float64)


def check(q, pages, page, table, lens, scale):
    """kv4_attention of q [sequences, heads, d] within the bound above."""
    dtype, d = q.dtype, q.shape[-1]
    group = q.shape[1] // pages.shape[1]
    got = kv4_attention(q.cuda(), KV4Cache(pages.cuda(), page, d), table.cuda(), lens.cuda(), scale=scale).double().cpu().numpy()
    step = torch.finfo(dtype).eps / 2
    for b, n in enumerate(lens.tolist()):
        k, v, _ = O.stored(pages, page, d, table, b, n)
        for h in range(q.shape[1]):
            x, kh, vh = (a.astype(np.float64) for a in (q[b, h].double().numpy(), k[:, h // group], v[:, h // group]))
            s = scale * (kh @ x)
            p = np.exp(s - s.max())
            p /= p.sum()
            sk, sv = (_scales(pages, d, table, page, b, n, h // group, i) for i in (False, True))
            top = (p * sv).max()
            score = (d + 16) * 2.0 ** -24 * scale * 30 * sk.max() * np.abs(x).sum()
            share = (2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11) + 2 * score + 2.0 ** -20
            want, mag = p @ vh, p @ np.abs(vh)
            tol = step * np.abs(want) + share * mag + ((n / 4 + 16) * 2.0 ** -24 * 30 + n * 2.0 ** -31 * 15) * top
            if dtype == torch.float16:
                tol = tol + 2.0 ** -25                                      # an output below 2^-14
            diff = np.abs(got[b, h] - want)
            assert np.isfinite(got[b, h]).all() and (diff <= tol).all(), (b, h, float((diff / tol).max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("small,large", [(2.0 ** -4, 2.0 ** 36), (2.0 ** -30, 2.0 ** 10), (2.0 ** -60, 2.0 ** 60)])
def test_peak_on_a_tiny_value(hip, dtype, small, large):
    """The peak at each place of a lane's eight tokens, in early and late blocks."""
    peaks = [0, 1, 2, 3, 16, 18, 21, 31, 32, 50, 70, 95, 99]
    d, page, n = 64, 32, 100
    g = torch.Generator().manual_seed(3)
    k = torch.randn(len(peaks) * n, 1, d, generator=g) * 0.05
    v = torch.randn(len(peaks) * n, 1, d, generator=g) * large
    for b, at in enumerate(peaks):
        k[b * n + at] = 0
        k[b * n + at, 0, 0] = 150.0                                         # 150 nats above the others
        v[b * n + at] *= small / large
    pages, table, lens = _pages([n] * len(peaks), k, v, page)
    q = torch.zeros(len(peaks), 2, d)
    q[..., 0], q[:, 1, 5] = 1.0, 0.25
    check(q.to(dtype), pages, page, table, lens, 1.0)
