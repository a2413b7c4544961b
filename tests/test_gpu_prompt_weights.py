"""The rounded weights of prompt attention are what its row sums count, so that their rounding cancels where values agree.

With every visible value equal to v, an output is (sum w) v / sum w for the same w above and below: fp32 roundings alone, (n + 4) of
2^-24 for the products' sums, n for the row's, 3 for the division: less than a quarter of a step of 2^-11 for n < 1000 rows, so v comes
out as it is."""
import pytest
import torch

from crispybits_kernels import prompt_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [40, 64, 80, 128, 256])
@pytest.mark.parametrize("lens", [[1] * 600, [2, 3, 64, 65, 130, 300, 1, 33]])
def test_equal_values_come_out_as_they_are(hip, dtype, d, lens):
    g = torch.Generator().manual_seed(d)
    rows = sum(lens)
    q, k = (torch.randn(rows, h, d, generator=g).to(dtype) for h in (4, 2))
    v = torch.cat([torch.randn(1, 2, d, generator=g).expand(n, 2, d) for n in lens]).to(dtype)
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).int()
    got = prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), max(lens)).cpu()
    want = v.repeat_interleave(2, 1)
    assert torch.equal(got, want), float(((got - want).abs() > 0).float().mean())
