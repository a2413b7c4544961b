"""kv4_append over the whole range of magnitudes: every word equals the oracle's, whose zero points and codes are found in
64 bits.  Zero points are decided near a half by the product's fast quotient, which has to keep its bits down to the smallest
ranges (fp32 and bf16 vectors of 1e-23 and less)."""
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_append, kv4_read
from oracle import attention as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [128, 256])
def test_every_magnitude(hip, dtype, d):
    """64 vectors a power of 2^5 from 2^-149 to 2^125, keys and values."""
    page, each = 64, 64
    powers = range(-149, 126, 5)
    g = torch.Generator().manual_seed(d)
    rows = each * len(powers)
    scale = torch.tensor([2.0 ** p for p in powers], dtype=torch.float64).repeat_interleave(each)[:, None, None]
    k, v = ((torch.randn(rows, 1, d, generator=g).clamp(-3, 3).double() * scale).to(dtype) for _ in range(2))
    table = torch.arange(-(-rows // page), dtype=torch.int32)[None]
    lens, cu = torch.tensor([rows], dtype=torch.int32), torch.tensor([0, rows], dtype=torch.int32)
    pages = torch.zeros(table.shape[1], 1, O.kv4_page_words(d, page), dtype=torch.int32)
    cache = KV4Cache(pages.clone().cuda(), page, d)
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    kv4_append(cache, k.cuda(), v.cuda(), table.cuda(), lens.cuda(), cu.cuda())
    got = cache.pages.cpu()
    wrong = (got != pages).view(table.shape[1], page // 32, -1)
    assert not wrong.any(), f"{int(wrong.any(-1).sum())} of {wrong.shape[0] * wrong.shape[1]} blocks"
    for a, b in zip(kv4_read(cache, table.cuda(), lens.cuda(), cu.cuda(), rows, dtype), O.kv4_read(pages, page, d, table, lens, cu, rows, dtype)):
        assert torch.equal(a.cpu(), b)
