"""Causal attention over packed prompts on the GPU against the float64 oracle (oracle/attention.py).

Bound of an output: its own rounding; the rounding of each weight to the type (half a step; none in fp32), which moves it by that
share of sum p |v|; the fp32 sums of scores (D products of at most |q| |k|), which move every weight by twice that; the fp32
sums over the tokens; 2^-20 for the exponentials.  fp16 weights below 2^-14 of the largest are held to 2^-25 of it."""
import numpy as np
import pytest
import torch

from crispybits_kernels import prompt_attention
from oracle import attention as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _inputs(lens, hq, hkv, d, dtype, seed, tail=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    rows = sum(lens) + tail
    q, k, v = ((torch.randn(rows, h, d, generator=g) * s).to(dtype) for h, s in ((hq, size), (hkv, size), (hkv, 1.0)))
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)
    return q, k, v, cu


def _check(got, q, k, v, cu, scale=None):
    d, dtype = q.shape[-1], q.dtype
    s = d ** -0.5 if scale is None else scale
    want, mag = O.prompt64(q, k, v, cu, s)
    step = torch.finfo(dtype).eps / 2
    group = q.shape[1] // k.shape[1]
    tol = step * np.abs(want)
    for a, z in zip(cu.tolist(), cu.tolist()[1:]):
        if a == z:
            continue
        n = z - a
        kk = np.repeat(np.abs(k[a:z].double().numpy()).max(0), group, axis=0)            # [heads, d]
        score = (d + 8) * 2.0 ** -24 * s * (np.abs(q[a:z].double().numpy()) * kk[None]).sum(-1)
        vm = np.repeat(np.abs(v[a:z].double().numpy()).max(0), group, axis=0)
        share = (0.0 if dtype == torch.float32 else step) + 2 * score + (n + 16) * 2.0 ** -24 + 2.0 ** -20
        tol[a:z] += share[..., None] * mag[a:z] + (n * 2.0 ** -25 * vm[None] if dtype == torch.float16 else 0.0)
    diff = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(diff).all()
    assert (diff <= tol).all(), float((diff / np.maximum(tol, 1e-300)).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 128), (8, 2, 128), (5, 1, 80), (4, 2, 64), (2, 1, 96), (2, 2, 256), (3, 3, 8),
                                      (2, 1, 40), (2, 2, 112), (2, 2, 136), (1, 1, 184), (6, 2, 72)])
def test_packed(hip, dtype, hq, hkv, d):
    lens = [1, 2, 0, 63, 64, 65, 127, 128, 129, 0, 200, 31]
    q, k, v, cu = _inputs(lens, hq, hkv, d, dtype, 1, size=2.0)
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), max(lens))
    _check(got, q, k, v, cu)
    again = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda())           # max_seqlen left out
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long(hip, dtype):
    q, k, v, cu = _inputs([700, 1100], 2, 1, 128, dtype, 2)
    _check(prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 1100), q, k, v, cu)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_and_none(hip, dtype):
    q, k, v, cu = _inputs([1], 4, 2, 128, dtype, 3)
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda())
    want = v.repeat_interleave(2, 1)
    if dtype == torch.float32:
        # (w v)(1 / w) for a weight w in (1/2, 1]: three roundings, each at most 2^-24 of the value
        assert ((got.cpu() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs()).all()
    else:
        # a 16-bit w is off by at most half a step at its smallest mantissa, which v's own rounding takes back
        assert torch.equal(got.cpu(), want)
    e = prompt_attention(q[:0].cuda(), k[:0].cuda(), v[:0].cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert e.shape == (0, 4, 128)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sharp_flat_and_growing_scores(hip, dtype):
    """Softmax sharpened and flattened by the scale, and keys whose scores grow along the sequence so that the running
    reference moves at every tile."""
    q, k, v, cu = _inputs([333], 2, 2, 64, dtype, 4)
    for scale in (5.0, 1e-3):
        _check(prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), scale=scale), q, k, v, cu, scale)
    q[..., 0], k[..., 0] = 4.0, (torch.arange(333.0) / 4).to(dtype)[:, None]
    _check(prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda()), q, k, v, cu)
    k[..., 0] = -k[..., 0]
    _check(prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda()), q, k, v, cu)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(hip, dtype):
    """Views of one tensor of all heads, heads before rows, a base off 16 bytes, a transposed head."""
    d, lens = 64, [70, 30]
    q, k, v, cu = _inputs(lens, 4, 2, d, dtype, 5)
    want = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda())
    _check(want, q, k, v, cu)
    one = torch.cat([q, k, v], dim=1).cuda()
    assert torch.equal(prompt_attention(one[:, :4], one[:, 4:6], one[:, 6:], cu.cuda()), want)
    a, b, c = (x.transpose(0, 1).contiguous().cuda().transpose(0, 1) for x in (q, k, v))
    assert torch.equal(prompt_attention(a, b, c, cu.cuda()), want)
    flat = torch.cat([torch.zeros(1, dtype=dtype), q.reshape(-1)]).cuda()
    assert torch.equal(prompt_attention(flat[1:].view(q.shape), k.cuda(), v.cuda(), cu.cuda()), want)
    t = v.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    assert torch.equal(prompt_attention(q.cuda(), k.cuda(), t, cu.cuda()), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sequence(hip, dtype):
    """Rows behind the last sequence: zeros in a new output, left as they were in a given one; whatever they hold."""
    for tail in (1, 150, 400):
        q, k, v, cu = _inputs([40, 90], 2, 1, 80, dtype, 6, tail=tail)
        for x in (q, k, v):
            x[130:] = float("nan")
        got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 90)
        assert not got[130:].any()
        out = torch.full_like(got, 3.0)
        assert prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), 90, out=out) is out
        assert torch.equal(out[:130], got[:130]) and (out[130:] == 3.0).all()
        _check(got[:130], q[:130], k[:130], v[:130], cu)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("where", [5, 64, 100, 127, 199])
def test_masked_places_take_no_part(hip, dtype, where):
    """Infinities and NaN in a token's key and value: rows before it are what they would be without, rows that see it
    have what the values give."""
    q, k, v, cu = _inputs([200], 2, 2, 80, dtype, 7)
    clean = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda())
    for kk, vv in ((float("nan"), 1.0), (1.0, float("nan")), (1.0, float("inf")), (float("inf"), float("-inf"))):
        k2, v2 = k.clone(), v.clone()
        k2[where, 0, 3] *= kk
        v2[where, :, 5], v2[where, 1, 77] = vv, -vv
        got = prompt_attention(q.cuda(), k2.cuda(), v2.cuda(), cu.cuda())
        assert torch.equal(got[:where], clean[:where])
        assert torch.isfinite(got[:where]).all()
        if kk == 1.0 and vv != 1.0:
            assert not torch.isfinite(got[where:, :, 5]).any() and not torch.isfinite(got[where:, 1, 77]).any()
            others = [i for i in range(80) if i not in (5, 77)]
            assert torch.equal(got[where:][..., others], clean[where:][..., others])
            if vv == float("inf"):
                assert (got[where:, :, 5] == float("inf")).all() and (got[where:, 1, 77] == float("-inf")).all()
        if kk != kk:
            assert torch.isnan(got[where:, 0]).all()


def test_captured_and_replayed(hip):
    """Two graphs of the call replayed with new inputs and lengths, eager work between."""
    g = torch.Generator().manual_seed(8)
    bufs = [[torch.zeros(300, h, 64, dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2)] for _ in range(2)]
    cus = [torch.zeros(4, dtype=torch.int32, device="cuda") for _ in range(2)]
    graphs, outs = [], []
    for b, cu in zip(bufs, cus):
        prompt_attention(*b, cu, 300)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(prompt_attention(*b, cu, 300))
        graphs.append(gr)
    for lens in ([100, 0, 200], [300, 0, 0], [1, 2, 3]):
        new = [torch.randn(300, h, 64, generator=g).bfloat16().cuda() for h in (4, 2, 2)]
        cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
        for b, c in zip(bufs, cus):
            for x, y in zip(b, new):
                x.copy_(y)
            c.copy_(cu)
        want = prompt_attention(*new, cu, 300)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
