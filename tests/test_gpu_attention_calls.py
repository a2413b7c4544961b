"""Calls of the attention ops as programs make them: refusals that name the argument, shared pages, calls without
arrival counters, several streams at once, a whole serving loop of packed projections, cache and attention."""
import numpy as np
import pytest
import torch

from crispybits_kernels import (KV4Cache, fused_qkv, kv4_append, kv4_attention, kv4_read, packed_linear, permute_for_rope,
                                prompt_attention)
from crispybits_kernels.io import from_packed_dict
from crispybits_kernels.reference import pack_linear_dict
from oracle import attention as O

pytestmark = pytest.mark.gpu


def _setup(lens=(40, 3), hkv=2, d=64, page=32, seed=0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n)
        at += n
    cache = KV4Cache.empty(at, hkv, d, page)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda()
    k, v = (torch.randn(sum(lens), hkv, d, generator=g).to(dtype).cuda() for _ in range(2))
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    kv4_append(cache, k, v, table.cuda(), ln, cu)
    return cache, table.cuda(), ln, cu, k, v


def test_refusals(hip):
    cache, table, ln, cu, k, v = _setup()
    q = torch.randn(2, 4, 64, device="cuda").half()

    def bad(match, f, *a, error=RuntimeError, **kw):
        with pytest.raises(error, match=match):
            f(*a, **kw)

    bad("one row per sequence", kv4_append, cache, k, v, table, ln)
    bad("one shape and dtype", kv4_append, cache, k, v.float(), table, ln, cu)
    bad("k and v must be", kv4_append, cache, k[:, :1], v[:, :1], table, ln, cu)
    bad("one more entry", kv4_append, cache, k, v, table, ln, cu[:2])
    bad("block_table must be", kv4_append, cache, k, v, table.long(), ln, cu)
    bad("block_table must be on the same device", kv4_append, cache, k, v, table.cpu(), ln, cu)
    bad("one row per sequence", kv4_append, cache, k, v, table[:1], ln, cu)
    bad("have 1152 words", kv4_append, KV4Cache(cache.pages, 64, 64), k, v, table, ln, cu)
    bad("page_size a power of two", kv4_append, KV4Cache(cache.pages, 48, 64), k, v, table, ln, cu)
    bad("fp16/bf16/fp32", kv4_append, cache, k.double(), v.double(), table, ln, cu)
    bad("no backward", kv4_append, cache, k.clone().requires_grad_(), v, table, ln, cu)
    bad("q must be", kv4_attention, q[:1], cache, table, ln)
    bad("q must be", kv4_attention, q[..., :32], cache, table, ln)
    bad("multiple of kv_heads", kv4_attention, q[:, :3], cache, table, ln)
    bad("scale must be", kv4_attention, q, cache, table, ln, scale=0.0)
    bad("scale must be", kv4_attention, q, cache, table, ln, scale=-1.0)
    bad("out must be", kv4_attention, q, cache, table, ln, out=torch.empty(2, 4, 64, device="cuda"))
    bad("overlaps an input", kv4_attention, q, cache, table, ln, out=q)
    bad("no backward", kv4_attention, q.clone().requires_grad_(), cache, table, ln)
    bad("dtype must be", kv4_read, cache, table, ln, cu, 43, torch.int32)
    bad("one dtype", prompt_attention, k, k, v.float(), cu)
    bad("k and v must be", prompt_attention, k, k[:-1], v[:-1], cu)
    bad("head_dim must be", prompt_attention, k[..., :12], k[..., :12], v[..., :12], cu)
    bad("cu_seqlens must be", prompt_attention, k, k, v, cu.long())
    bad("max_seqlen must be", prompt_attention, k, k, v, cu, 0)
    bad("overlaps an input", prompt_attention, k, k, v, cu, out=v)
    bad("no backward", prompt_attention, k, k, v.clone().requires_grad_(), cu)
    with torch.no_grad():                                      # a model's own tensors, outside of training
        prompt_attention(k.clone().requires_grad_(), k, v, cu)
    torch.cuda.synchronize()


def test_shared_pages(hip):
    """Two sequences over one prefix's pages, and one sequence twice."""
    cache, table, ln, _, _, _ = _setup((64, 40))
    both = torch.stack([table[0], table[0], torch.tensor([0, 2], device="cuda", dtype=torch.int32)])
    n = torch.tensor([64, 64, 50], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    q[1] = q[0]
    got = kv4_attention(q, cache, both, n)
    assert torch.equal(got[0], got[1])
    want, _ = O.attention64(q[:, None].cpu(), cache.pages.cpu(), 32, 64, both.cpu(), n.cpu(), 64 ** -0.5)
    np.testing.assert_allclose(got.double().cpu().numpy(), want[:, 0], atol=4e-3)


def test_without_counters(hip):
    """On the per-thread default stream there are no arrival counters: the second launch gives the same bits."""
    cache, table, ln, _, _, _ = _setup((3000, 700, 9000), 2, 128, 64, seed=2)
    q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(3)).half().cuda()
    want = kv4_attention(q, cache, table, ln)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.ExternalStream(2)):      # hipStreamPerThread
        got = kv4_attention(q, cache, table, ln)
        torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_two_streams_at_once(hip):
    """Calls on two streams over one cache, many times: each has its own partials and counters."""
    cache, table, ln, _, _, _ = _setup((5000, 300), 2, 128, 64, seed=4)
    qs = [torch.randn(2, 4, 128, generator=torch.Generator().manual_seed(5 + i)).half().cuda() for i in range(2)]
    want = [kv4_attention(q, cache, table, ln) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(kv4_attention(qs[i], cache, table, ln))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_serving_loop(hip, dtype):
    """Packed projections, rotation, cache and attention as a decoder layer runs them: packed prompts, then decode steps
    from a captured graph, against float64 attention over what the cache holds."""
    hidden, hq, hkv, d = 512, 8, 2, 64
    lens, page, steps = [70, 1, 33], 32, 4
    g = torch.Generator().manual_seed(6)
    ws = [from_packed_dict(pack_linear_dict(torch.randn(n, hidden, generator=g) * 0.05, 4, 128, None, dtype), "cuda", dtype)
          for n in (hq * d, hkv * d, hkv * d, hidden)]
    wq, wk, wv, wo = permute_for_rope(ws[0], d), permute_for_rope(ws[1], d), ws[2], ws[3]
    table = torch.arange(3 * 4, dtype=torch.int32, device="cuda").view(3, 4)
    cache = KV4Cache.empty(12, hkv, d, page)
    inv = 10000.0 ** (-torch.arange(0, d, 2).float() / d)

    def tables(pos):
        a = torch.cat([pos[:, None].float() * inv] * 2, dim=1)
        return a.cos().to(dtype).cuda(), a.sin().to(dtype).cuda()

    rows = sum(lens)
    x = torch.randn(rows, hidden, generator=g).to(dtype).cuda()
    pos = torch.cat([torch.arange(n) for n in lens])
    q, k, v = fused_qkv(x, wq, wk, wv, rope=(*tables(pos), d))
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32).cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    q, k, v = q.view(rows, hq, d), k.view(rows, hkv, d), v.view(rows, hkv, d)
    kv4_append(cache, k, v, table, n, cu)
    o = prompt_attention(q, k, v, cu, max(lens))
    y = packed_linear(o.view(rows, hq * d), wo)
    want, _ = O.prompt64(q.cpu(), k.cpu(), v.cpu(), cu.cpu(), d ** -0.5)
    tol = 1e-2 if dtype == torch.bfloat16 else 2e-3
    assert np.abs(o.double().cpu().numpy() - want).max() <= tol * np.abs(want).max()
    assert torch.isfinite(y).all()

    x1 = torch.zeros(3, hidden, dtype=dtype, device="cuda")
    cs = [torch.zeros(3, d, dtype=dtype, device="cuda") for _ in range(2)]

    def step():
        q, k, v = fused_qkv(x1, wq, wk, wv, rope=(cs[0], cs[1], d))
        n.add_(1)
        kv4_append(cache, k.view(3, hkv, d), v.view(3, hkv, d), table, n)
        o = kv4_attention(q.view(3, hq, d), cache, table, n)
        return q, o, packed_linear(o.view(3, hq * d), wo)

    keep, held = n.clone(), cache.pages.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q1, o1, y1 = step()
    n.copy_(keep)
    cache.pages.copy_(held)
    for i in range(steps):
        x1.copy_(torch.randn(3, hidden, generator=g).to(dtype))
        for a, b in zip(cs, tables(torch.tensor(lens) + i)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert n.tolist() == [m + i + 1 for m in lens]
        want, _ = O.attention64(q1.view(3, 1, hq, d).cpu(), cache.pages.cpu(), page, d, table.cpu(), n.cpu(), d ** -0.5)
        assert np.abs(o1.double().cpu().numpy() - want[:, 0]).max() <= tol * np.abs(want).max()
        assert torch.isfinite(y1).all()
