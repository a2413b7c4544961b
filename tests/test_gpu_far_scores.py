"""Scores far from zero, of either sign, up to the edge of fp32: softmax of finite scores is finite.

Keys take few values and queries one, so that scores are exact products with ties, and different scores lie so far apart that
a row's softmax is even over the visible tokens of its largest score.  Bound of an output: its own rounding, the weights' (half a step
of the type), 2^-20 for the exponentials and the fp32 sums."""
import numpy as np
import pytest
import torch

from crispybits_kernels import prompt_attention
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
