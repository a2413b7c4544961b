"""Prompt attention where a few tokens hold nearly all of the weight and very many others share the rest.

Bound of an output as in test_gpu_prompt_attention.py, but for the smallest fp16 weights: the largest weight of a row stands
at 2^6 at least, so the half step of 2^-25 that a denormal one may lose is 2^-31 of it.  An fp16 output below 2^-14 is rounded by
half a step of 2^-24."""
import numpy as np
import pytest
import torch

from crispybits_kernels import prompt_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu


def _rows_are_right(got, q, k, v, rows, scale):
    dtype, n_heads = q.dtype, q.shape[1]
    step = torch.finfo(dtype).eps / 2
    for r in rows:
        for h in range(n_heads):
            a, b, c = (t[:r + 1, h].double().numpy() for t in (q, k, v))
            want, mag = O.softmax_rows(a[r:], b, c, np.ones((1, r + 1), bool), scale)
            score = (q.shape[2] + 8) * 2.0 ** -24 * scale * np.abs(a[r]) @ np.abs(b).max(0)
            share = (0.0 if dtype == torch.float32 else step) + 2 * score + (r + 17) * 2.0 ** -24 + 2.0 ** -20
            tol = step * np.abs(want) + share * mag
            if dtype == torch.float16:
                tol = tol + (r + 1) * 2.0 ** -31 * np.abs(c).max(0) + 2.0 ** -25
            diff = np.abs(got[r, h].double().cpu().numpy() - want[0])
            assert (diff <= tol[0]).all(), (r, h, float((diff / tol[0]).max()), float(got[r, h, 0]), float(want[0, 0]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_first_token_and_flat_tail(hip, dtype, d):
    """The first token's score lies 17.5 above all others', 2^-25.2 as a weight: 30,000 of them are 7.5e-4 of the whole.  In
    head 0 the first value is zero and the others are one, in head 1 all are one, head 2 has any."""
    n = 30000
    g = torch.Generator().manual_seed(d)
    q, k, v = (torch.zeros(n, 3, d) for _ in range(3))
    q[..., 0], k[0, :, 0] = 3.5, 5.0
    q[..., 1:8] = torch.randn(n, 3, 7, generator=g)
    k[..., 1:8] = torch.randn(n, 3, 7, generator=g) * 0.05
    v[1:, 0], v[:, 1] = 1.0, 1.0
    v[:, 2] = torch.randn(n, d, generator=g)
    q, k, v = (t.to(dtype) for t in (q, k, v))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu, n, scale=1.0)
    _rows_are_right(got, q, k, v, (0, 1, 63, 64, 700, 4095, n // 2, n - 1), 1.0)
