"""The paged 4-bit cache on the GPU against the float64 oracle (oracle/attention.py): append word by word, read bit
by bit, attention within the bounds that the arithmetic allows.

Bounds of attention (``_bound``).  Codes, zero points and (fp16 / bf16) q are exact in the products, so an output is
off by: its own rounding; the rounding of each weight to fp16 (half a step: 2^-11; fp32: two terms, 2^-22), which moves it by
that share of sum p |v|; the fp32 sums of scores (D products and the two terms of a zero point, each at most 15 s |q|), which
move every weight by twice that; and the fp32 sums over the tokens (codes and zero points apart, each at most
15 s p), about eight roundings for each product of 32 tokens."""
import numpy as np
import pytest
import torch

from crispybits_kernels import KV4Cache, kv4_append, kv4_attention, kv4_read
from oracle import attention as O

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _cumulative(n):
    return [0] + list(np.cumsum(n))


def _case(lens, hkv, d, page, seed, dtype=torch.float16, spread=1.0):
    """(cache on the GPU, the oracle's pages, table, lens) of sequences with random tokens, pages out of order in a
    pool whose unused words are junk."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-n // page)) for n in lens]
    pool = sum(need) + 2
    ids = torch.randperm(pool, generator=g).int()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    words = O.kv4_page_words(d, page)
    pages = torch.randint(-2 ** 31, 2 ** 31 - 1, (pool, hkv, words), generator=g, dtype=torch.int64).int()
    ln = torch.tensor(lens, dtype=torch.int32)
    cu = torch.tensor(_cumulative([max(n, 0) for n in lens]), dtype=torch.int32)
    rows = int(cu[-1])
    k, v = ((torch.randn(rows, hkv, d, generator=g) * torch.exp(spread * torch.randn(rows, hkv, 1, generator=g))).to(dtype)
            for _ in range(2))
    O.kv4_append(pages, page, d, k, v, table, ln, cu)
    return KV4Cache(pages.clone().cuda(), page, d), pages, table, ln


def _bound(q, pages, page, d, table, lens, scale, out, mag):
    """The largest error allowed, elementwise [seqs, t, heads, D]."""
    dtype = q.dtype
    step = torch.finfo(dtype).eps / 2
    weight = 2.0 ** -22 if dtype == torch.float32 else 2.0 ** -11
    group = q.shape[2] // pages.shape[1]
    tol = step * np.abs(out)
    qa = np.abs(q.double().cpu().numpy()).sum(-1)                       # [seqs, t, heads]
    words = pages.numpy().view(np.uint32).reshape(pages.shape[0], pages.shape[1], -1, O._block_words(d))
    ns = -(-d // 32)
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        blocks = [(int(table[b, i // page]), i % page // 32, i % 32) for i in range(n)
                  if 0 <= table[b, i // page] < pages.shape[0]]
        sk = np.array([words[p, :, x, 256 * ns + t] for p, x, t in blocks]).view(np.float32)      # [n, hkv]
        sv = np.array([words[p, :, x, 256 * ns + 32 + t] for p, x, t in blocks]).view(np.float32)
        ks, vs = (np.repeat(s.max(0), group)[None, :] for s in (sk, sv))
        score = (d + 16) * 2.0 ** -24 * scale * 30 * ks * qa[b]
        if dtype == torch.float32:
            score = score + 2.0 ** -22 * scale * 15 * ks * qa[b]
        share = weight + 2 * score + 2.0 ** -20
        sums = (n / 4 + 16) * 2.0 ** -24 * 30 * vs + n * 2.0 ** -28 * 15 * vs
        tol[b] += share[..., None] * mag[b] + np.broadcast_to(sums, share.shape)[..., None]
    return tol


def _check(q, cache, pages, table, lens, scale=None, out=None):
    d = cache.head_dim
    s = d ** -0.5 if scale is None else scale
    got = kv4_attention(q.cuda(), cache, table.cuda(), lens.cuda(), scale=scale, out=out)
    q4 = q if q.dim() == 4 else q.unsqueeze(1)
    want, mag = O.attention64(q4, pages, cache.page_size, d, table, lens, s)
    tol = _bound(q4, pages, cache.page_size, d, table, lens, s, want, mag)
    diff = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert np.isfinite(diff).all()
    assert (diff <= tol).all(), float((diff / np.maximum(tol, 1e-300)).max())
    return got


# ------------------------------------------------------------------------------------- append and read

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,hkv,page", [(128, 2, 64), (80, 3, 32), (64, 5, 128), (8, 1, 32), (72, 2, 64), (136, 1, 32),
                                        (256, 2, 64), (200, 1, 32)])
def test_append_is_exact(hip, dtype, d, hkv, page):
    """Prompts behind prefixes of odd lengths: every word of the pool equals the oracle's, the words of other
    tokens and pages untouched."""
    held, new = [0, 5, 31, 33, 63, 7], [40, 1, 1, 95, 2, 0]
    cache, pages, table, lens = _case([h + n for h, n in zip(held, new)], hkv, d, page, 1, dtype)
    g = torch.Generator().manual_seed(2)
    cu = torch.tensor(_cumulative(new), dtype=torch.int32)
    k, v = ((torch.randn(int(cu[-1]), hkv, d, generator=g) * 3).to(dtype) for _ in range(2))
    k[0], v[1] = 0, 0                                                   # all zeros
    k[2, 0] = k[2, 0].abs() + 100                                       # far from zero, one sign
    v[3, 0, :] = torch.linspace(-1, 1, d).to(dtype)                     # symmetric: a tie for the zero point
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    kv4_append(cache, k.cuda(), v.cuda(), table.cuda(), lens.cuda(), cu.cuda())
    assert torch.equal(cache.pages.cpu(), pages)
    got = kv4_read(cache, table.cuda(), lens.cuda(), cu.cuda(), int(cu[-1]), dtype)
    want = O.kv4_read(pages, page, d, table, lens, cu, int(cu[-1]), dtype)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_one_token(hip, dtype):
    """A decode step's rows: no cu_seqlens, an idle slot, a sequence whose page is missing, views of one tensor."""
    d, hkv, page = 128, 4, 64
    cache, pages, table, lens = _case([1, 64, 65, 0, 130, 127], hkv, d, page, 3, dtype)
    table[4, 2] = -1
    g = torch.Generator().manual_seed(4)
    both = torch.randn(6, 3 * hkv, d, generator=g).to(dtype)
    k, v = both[:, hkv:2 * hkv], both[:, 2 * hkv:]
    O.kv4_append(pages, page, d, k, v, table, lens)
    dev = both.cuda()
    kv4_append(cache, dev[:, hkv:2 * hkv], dev[:, 2 * hkv:], table.cuda(), lens.cuda())
    assert torch.equal(cache.pages.cpu(), pages)
    for a, b in zip(kv4_read(cache, table.cuda(), lens.cuda(), dtype=dtype), O.kv4_read(pages, page, d, table, lens, None, 6, dtype)):
        assert torch.equal(a.cpu(), b)


def test_append_strided_and_unaligned(hip):
    """Rows that the kernels cannot step through in 16-byte pieces are copied first: the same words."""
    d, hkv, page = 64, 2, 32
    g = torch.Generator().manual_seed(5)
    base = torch.randn(20 * hkv * d + 1, generator=g).half()
    k, v = base[1:].view(20, hkv, d), torch.randn(20, d, hkv, generator=g).half().transpose(1, 2)
    cache, pages, table, lens = _case([20], hkv, d, page, 6)
    O.kv4_append(pages, page, d, k, v, table, lens, torch.tensor([0, 20], dtype=torch.int32))
    dev = base.cuda()
    kv4_append(cache, dev[1:].view(20, hkv, d), v.transpose(1, 2).contiguous().cuda().transpose(1, 2), table.cuda(), lens.cuda(),
               torch.tensor([0, 20], dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.pages.cpu(), pages)


def test_append_borders_and_extremes(hip):
    """Values a hair from the borders between codes, the smallest and largest magnitudes, values that are not finite."""
    d, page = 128, 32
    g = torch.Generator().manual_seed(7)
    x = torch.randn(60, 1, d, generator=g)
    x[:20, :, 0], x[:20, :, 1] = 7.5, 0.0                               # steps of one half: ties at quarters
    x[:20, :, 2:] = torch.randint(0, 31, (20, 1, d - 2), generator=g) * 0.25
    x[20:40] = x[:20] * (1 + 2.0 ** -23) ** torch.randint(-3, 4, (20, 1, d), generator=g)
    x[40] *= 1e-37
    x[41] *= 1e38 / 5
    x[42] *= 1e-42
    x[43, 0, 5], x[44, 0, 6], x[45, 0, 7] = float("inf"), float("-inf"), float("nan")
    cache, pages, table, lens = _case([60], 1, d, page, 8, torch.float32)
    cu = torch.tensor([0, 60], dtype=torch.int32)
    O.kv4_append(pages, page, d, x, x.flip(0), table, lens, cu)
    kv4_append(cache, x.cuda(), x.flip(0).cuda(), table.cuda(), lens.cuda(), cu.cuda())
    assert torch.equal(cache.pages.cpu(), pages)
    k, _ = kv4_read(cache, table.cuda(), lens.cuda(), cu.cuda(), 60, torch.float32)
    assert torch.isnan(k[43:46]).all() and torch.isfinite(k[:43]).all() and torch.isfinite(k[46:]).all()


def test_rows_of_no_sequence(hip):
    """Rows before the first sequence and behind the last: not stored, read as zeros."""
    d, hkv, page = 96, 2, 32
    cache, pages, table, lens = _case([50, 40], hkv, d, page, 9)
    cu = torch.tensor([37, 77, 117], dtype=torch.int32)
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(200, hkv, d, generator=g).half() for _ in range(2))
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    kv4_append(cache, k.cuda(), v.cuda(), table.cuda(), lens.cuda(), cu.cuda())
    assert torch.equal(cache.pages.cpu(), pages)
    got = kv4_read(cache, table.cuda(), lens.cuda(), cu.cuda(), 200)
    want = O.kv4_read(pages, page, d, table, lens, cu, 200, torch.float16)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
        assert not a[:37].any() and not a[117:].any()


def test_many_sequences(hip):
    """More sequences than a wave looks at at once, of zero to three new tokens."""
    d, hkv, page = 64, 1, 32
    new = [i % 4 for i in range(150)]
    cache, pages, table, lens = _case([n + 30 for n in new], hkv, d, page, 11)
    cu = torch.tensor(_cumulative(new), dtype=torch.int32)
    g = torch.Generator().manual_seed(12)
    k, v = (torch.randn(int(cu[-1]), hkv, d, generator=g).half() for _ in range(2))
    O.kv4_append(pages, page, d, k, v, table, lens, cu)
    kv4_append(cache, k.cuda(), v.cuda(), table.cuda(), lens.cuda(), cu.cuda())
    assert torch.equal(cache.pages.cpu(), pages)


# ------------------------------------------------------------------------------------- attention

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,page", [(4, 4, 128, 64), (8, 2, 128, 32), (5, 1, 80, 64), (4, 2, 64, 128), (16, 1, 96, 32),
                                           (2, 2, 256, 64), (3, 3, 8, 32), (4, 2, 136, 32), (6, 3, 200, 32)])
def test_attention_one_token(hip, dtype, hq, hkv, d, page):
    lens = [1, 2, 31, 32, 33, 0, 100, 161, 300]
    cache, pages, table, ln = _case(lens, hkv, d, page, 20, dtype)
    q = (torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(21)) * 2).to(dtype)
    got = _check(q, cache, pages, table, ln)
    assert not got[5].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,hq,hkv", [(2, 4, 4), (4, 8, 2), (5, 8, 1), (7, 3, 3), (33, 2, 1)])
def test_attention_new_tokens(hip, dtype, t, hq, hkv):
    """Several new tokens a sequence, each seeing up to itself; sequences shorter than t have rows that see nothing."""
    lens = [t, t + 1, 40, 97, 1, 0, 250]
    cache, pages, table, ln = _case(lens, hkv, 64, 32, 22, dtype)
    q = torch.randn(len(lens), t, hq, 64, generator=torch.Generator().manual_seed(23)).to(dtype)
    got = _check(q, cache, pages, table, ln)
    if t > 1:
        assert not got[4, :t - 1].any() and not got[5].any()


def test_attention_long_and_split(hip):
    """One sequence over many workgroups, and one next to it that fits one."""
    cache, pages, table, ln = _case([5000, 100], 2, 128, 64, 24)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(25)).half()
    a = _check(q, cache, pages, table, ln)
    b = kv4_attention(q.cuda(), cache, table.cuda(), ln.cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many_sequences(hip, dtype):
    """More sequences than a wave looks at at once, empty ones and long ones among them: units whole, cut once and cut often."""
    lens = [(7 * i) % 45 for i in range(150)]
    lens[3], lens[70], lens[149] = 1500, 700, 900
    cache, pages, table, ln = _case(lens, 1, 64, 32, 40, dtype)
    q = torch.randn(150, 2, 64, generator=torch.Generator().manual_seed(41)).to(dtype)
    got = _check(q, cache, pages, table, ln)
    assert not got[0].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_row_tiles_cut(hip, dtype):
    """Several tiles of query rows a head, the last one part full, over sequences long enough to be cut."""
    cache, pages, table, ln = _case([2100, 50, 640], 2, 128, 64, 42, dtype)
    q = torch.randn(3, 9, 8, 128, generator=torch.Generator().manual_seed(43)).to(dtype)
    _check(q, cache, pages, table, ln)


def test_attention_scales_and_magnitudes(hip):
    """Sharp and flat softmax, scales of tokens spread over orders of magnitude, tiny and huge values."""
    for spread, size, scale in ((0.1, 1.0, 3.0), (3.0, 1.0, 0.02), (1.0, 1e-6, 1e5), (1.0, 1e4, 1e-7)):
        g = torch.Generator().manual_seed(26)
        cache, pages, table, ln = _case([200, 77], 2, 128, 32, 27, torch.float32, spread)
        cu = torch.tensor([0, 200, 277], dtype=torch.int32)
        k, v = (torch.randn(277, 2, 128, generator=g) * size * torch.exp(spread * torch.randn(277, 2, 1, generator=g)) for _ in range(2))
        O.kv4_append(pages, 32, 128, k, v, table, ln, cu)
        cache.pages.copy_(pages)
        for dtype in DTYPES:
            if dtype == torch.float16 and size != 1.0:
                continue
            _check(torch.randn(2, 4, 128, generator=g).to(dtype), cache, pages, table, ln, scale)


def test_attention_masked_junk(hip):
    """Stale words behind the last token (NaN and infinite scales), missing pages inside and behind the table's use, a
    length beyond the table: none takes part.  NaN in a visible token reaches the rows that see it, and only those."""
    d, hkv, page = 128, 2, 32
    cache, pages, table, ln = _case([70, 90, 64], hkv, d, page, 28)
    ns = 4
    w = pages.view(pages.shape[0], hkv, 1, -1)
    bad = np.array([0x7FC00003, 0x7F800000, 0xFF800000], dtype=np.uint32).view(np.int32)
    for b, n in ((0, 70), (1, 90)):
        for t in range(n % 32, 32):
            w[table[b, n // 32], :, 0, 256 * ns + t] = int(bad[t % 3])
            w[table[b, n // 32], :, 0, 256 * ns + 32 + t] = int(bad[(t + 1) % 3])
    cache.pages.copy_(pages)
    q = torch.randn(3, 3, 4, d, generator=torch.Generator().manual_seed(29)).half()
    _check(q, cache, pages, table, ln)
    hole = table.clone()
    hole[1, 1] = -1
    hole[2, 0] = pages.shape[0]
    _check(q, cache, pages, hole, ln)
    longer = ln.clone()
    longer[2] = 64 + 4 * 32                                            # behind the table's width
    want, _ = O.attention64(q, pages, page, d, table, longer, d ** -0.5)
    got = kv4_attention(q.cuda(), cache, table.cuda(), longer.cuda())
    assert torch.isfinite(got).all()
    np.testing.assert_allclose(got[2].double().cpu().numpy(), want[2], atol=2e-2)
    # the newest token of sequence 0 is NaN: query 2 of 3 sees it, queries 0 and 1 do not
    w[table[0, 2], 0, 0, 256 * ns + 32 + 69 % 32] = int(bad[0])
    cache.pages.copy_(pages)
    got = kv4_attention(q.cuda(), cache, table.cuda(), ln.cuda())
    assert torch.isnan(got[0, 2, :2]).all() and torch.isfinite(got[0, :2]).all() and torch.isfinite(got[0, 2, 2:]).all()


def test_attention_into_out_and_shapes(hip):
    cache, pages, table, ln = _case([33, 10], 2, 64, 32, 30)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(31)).half()
    out = torch.full((2, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    got = _check(q, cache, pages, table, ln, out=out)
    assert got is out
    e = kv4_attention(q[:0].cuda(), cache, table[:0].cuda(), ln[:0].cuda())
    assert e.shape == (0, 4, 64)
    strided = torch.randn(2, 64, 4, generator=torch.Generator().manual_seed(32)).half().transpose(1, 2)
    _check(strided, cache, pages, table, ln)


def test_large_pool(hip):
    """Pages past 2^32 bytes into the pool."""
    d, hkv, page = 128, 8, 256
    words = O.kv4_page_words(d, page)
    n = 2 ** 33 // (hkv * words * 4)
    pages = torch.zeros(n + 1, hkv, words, dtype=torch.int32, device="cuda")
    cache = KV4Cache(pages, page, d)
    table = torch.tensor([[n, n - 1]], dtype=torch.int32)
    ln = torch.tensor([300], dtype=torch.int32)
    g = torch.Generator().manual_seed(33)
    k, v = (torch.randn(300, hkv, d, generator=g).half() for _ in range(2))
    cu = torch.tensor([0, 300], dtype=torch.int32)
    kv4_append(cache, k.cuda(), v.cuda(), table.cuda(), ln.cuda(), cu.cuda())
    small = torch.zeros(2, hkv, words, dtype=torch.int32)
    st = torch.tensor([[1, 0]], dtype=torch.int32)
    O.kv4_append(small, page, d, k, v, st, ln, cu)
    assert torch.equal(pages[n - 1:].cpu(), small) and not pages[:n - 1].any()
    q = torch.randn(1, 8, d, generator=g).half()
    got = kv4_attention(q.cuda(), cache, table.cuda(), ln.cuda())
    _check(q, KV4Cache(small.cuda(), page, d), small, st, ln)
    assert torch.equal(got, kv4_attention(q.cuda(), KV4Cache(small.cuda(), page, d), st.cuda(), ln.cuda()))


def test_streams_graphs_and_growth(hip):
    """A captured decode step (lengths, append, attention) replayed as sequences grow, with eager work between the
    replays and on another stream; two graphs of it side by side."""
    d, hq, hkv, page, b = 128, 8, 2, 32, 3
    start = [40, 1, 2000]
    table_len = 80
    ids = torch.randperm(b * table_len, generator=torch.Generator().manual_seed(34)).int().view(b, table_len)
    caches = [KV4Cache.empty(b * table_len, hkv, d, page) for _ in range(3)]
    table = ids.cuda()
    g = torch.Generator().manual_seed(35)
    rows = sum(start)
    k0, v0 = (torch.randn(rows, hkv, d, generator=g).half().cuda() for _ in range(2))
    cu = torch.tensor(_cumulative(start), dtype=torch.int32, device="cuda")
    lens = [torch.tensor(start, dtype=torch.int32, device="cuda") for _ in range(3)]
    for c, n in zip(caches, lens):
        kv4_append(c, k0, v0, table, n, cu)
    x = [[torch.zeros(b, h, d, dtype=torch.float16, device="cuda") for h in (hq, hkv, hkv)] for _ in range(3)]

    def step(i):
        lens[i].add_(1)
        kv4_append(caches[i], x[i][1], x[i][2], table, lens[i])
        return kv4_attention(x[i][0], caches[i], table, lens[i])

    graphs, outs = [], []
    side = torch.cuda.Stream()
    for i in (1, 2):
        keep, held = lens[i].clone(), caches[i].pages.clone()
        with torch.cuda.stream(side):
            step(i)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(i))
        graphs.append(gr)
        lens[i].copy_(keep)
        caches[i].pages.copy_(held)
    for rep in range(5):
        new = [torch.randn(b, h, d, generator=g).half().cuda() for h in (hq, hkv, hkv)]
        for i in range(3):
            for a, s in zip(x[i], new):
                a.copy_(s)
        want = step(0)
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), rep
    assert torch.equal(caches[0].pages, caches[1].pages) and torch.equal(caches[0].pages, caches[2].pages)
