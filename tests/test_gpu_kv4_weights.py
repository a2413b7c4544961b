"""fp16 attention over the 4-bit cache holds its weights to 22 bits: where values cancel, an output is as exact as its own
rounding and the fp32 sums leave it.

Bound of an output, of sequences of a few tokens whose queries and keys have one value: its rounding (2^-11, at least half of 2^-24); each
weight's 2^-22, 2^-20 for the exponentials and twice the scores' error, each (d + 16) roundings of at most 30 s |q|; and the sums', 32
roundings of at most 30 p s' (as in test_gpu_kv4.py)."""
import numpy as np
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 80, 128, 256])
def test_values_that_cancel(hip, d):
    seqs, heads, n, page = 48, 4, 6, 32
    g = torch.Generator().manual_seed(d)
    k = torch.zeros(seqs * n, 1, d)
    k[..., 1] = torch.rand(seqs * n, 1, generator=g)
    v = torch.randn(seqs, 1, 1, d, generator=g) * torch.tensor([1.0, -1.0] * (n // 2)).view(1, n, 1, 1)
    v = v.reshape(seqs * n, 1, d).contiguous()
    table = torch.arange(seqs, dtype=torch.int32)[:, None].contiguous()
    lens, cu = torch.full((seqs,), n, dtype=torch.int32), torch.arange(0, (seqs + 1) * n, n, dtype=torch.int32)
    pages = torch.zeros(seqs, 1, O.kv4_page_words(d, page), dtype=torch.int32)
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    q = torch.zeros(seqs, heads, d)
    q[..., 1] = torch.tensor([0.25, 0.5, 1.0, 2.0])
    got = kv4_attention(q.half().cuda(), KV4Cache(pages.cuda(), page, d), table.cuda(), lens.cuda(), scale=1.0).double().cpu().numpy()
    worst = 0.0
    for b in range(seqs):
        kk, vv, _ = O.stored(pages, page, d, table, b, n)
        K, V = kk[:, 0].astype(np.float64), vv[:, 0].astype(np.float64)
        sk, sv = np.abs(K).max() / 7, np.abs(V).max() / 7                     # no scale is larger
        for h in range(heads):
            s = K @ q[b, h].double().numpy()
            p = np.exp(s - s.max())
            p /= p.sum()
            want, mag = p @ V, p @ np.abs(V)
            share = 2.0 ** -22 + 2.0 ** -20 + 2 * (d + 16) * 2.0 ** -24 * 30 * sk * float(q[b, h, 1])
            tol = np.maximum(2.0 ** -11 * np.abs(want), 2.0 ** -25) + share * mag + 32 * 2.0 ** -24 * 30 * p.max() * sv
            worst = max(worst, float((np.abs(got[b, h] - want) / tol).max()))
    assert worst <= 1.0, worst
