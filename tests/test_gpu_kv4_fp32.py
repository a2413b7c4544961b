"""fp32 attention over the 4-bit cache is as exact as fp32 allows: nothing is held in fewer bits.

Bound of an output, u = 2^-24, for sequences of at most 546 tokens (below that the whole parts of 2^11 x 15 n stay below 2^24, exact):
each weight is off by the score's roundings (its product with s, its sum's: 2 u |score|; queries held to 2^-34 of their largest value,
15 s D of them; the products of queries' lower terms, less), 2 u for the exponential and 2 u for its argument's, the sum of weights by n / 16
additions a lane and 10 more (a weight's error counts twice, in the sum too), and the output by eight roundings where two terms, four waves
and parts meet.  Weights times s' are held to 2^-30 of the largest (15 times for each token), and a matrix product
cuts terms 2^-26 below its largest, 2^-24 of the largest weight a product in all."""
import numpy as np
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("scale,size", [(None, 1.0), (0.02, 1.0), (0.5, 1.0), (None, 1e-5), (None, 1e6)])
def test_error_is_that_of_fp32(hip, d, scale, size):
    b, heads, group, n, page, u = 2, 2, 16, 500, 64, 2.0 ** -24
    scale = d ** -0.5 if scale is None else scale
    g = torch.Generator().manual_seed(d)
    k, v = torch.randn(b * n, heads, d, generator=g), torch.randn(b * n, heads, d, generator=g) * size
    q = torch.randn(b, heads * group, d, generator=g)
    need = -(-n // page)
    table = torch.arange(b * need, dtype=torch.int32).view(b, need)
    lens, cu = torch.full((b,), n, dtype=torch.int32), torch.arange(0, (b + 1) * n, n, dtype=torch.int32)
    pages = torch.zeros(b * need, heads, O.kv4_page_words(d, page), dtype=torch.int32)
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    got = kv4_attention(q.cuda(), KV4Cache(pages.cuda(), page, d), table.cuda(), lens.cuda(), scale=scale).double().cpu().numpy()
    worst = 0.0
    for i in range(b):
        kk, vv, _ = O.stored(pages, page, d, table, i, n)
        for h in range(heads * group):
            x, K, V = q[i, h].double().numpy(), kk[:, h // group].astype(np.float64), vv[:, h // group].astype(np.float64)
            s = scale * (K @ x)
            p = np.exp(s - s.max())
            p /= p.sum()
            want, mag = p @ V, p @ np.abs(V)
            sk, sv = (np.abs(a).max() / 7 for a in (K, V))                # no scale is larger: 15 steps over a range, zero inside
            score = 2 * u * np.abs(s).max() + d * 2.0 ** -34 * np.abs(x).max() * 15 * sk * scale
            tol = u * np.abs(want) + (2 * (score + 4 * u) + (n / 16 + 10 + 8) * u) * mag
            tol = tol + (n * 2.0 ** -30 * 15 + (n / 64 + 2) * u) * p.max() * sv
            diff = np.abs(got[i, h] - want)
            worst = max(worst, float((diff / tol).max()))
    assert worst <= 1.0, worst
