"""The attention operators whose speed counts, in their plain form and as a user's program calls them.

A case is a plain dict; ``listed()`` names the fixed ones, ``draw(rng)`` gives more of the same ranges.
``prepare`` makes the inputs on the GPU from a seed, ``run`` is one pass (elementary torch operations, or
with ``own`` the framework's calls), ``exact`` the same results in 64 bits from the definition, ``work``
the bytes and operations one pass cannot do without.

Kinds:
  prompt  causal attention over packed prompts of different lengths, grouped heads
  decode  attention of each sequence's newest token (or few tokens) over a paged cache held in 4 bits
  append  new tokens' keys and values into that cache, and read back as the values they stand for

The cache.  ``pages`` is int32 [pages, kv heads, page words]; token i of a sequence lies in page
``table[sequence, i // page]`` at slot i % page.  A vector x of a token and head is stored as 4-bit codes c
with a scale s and a zero point z, x = s (c - z).  The scale is a float whose low four mantissa bits hold
z.  Slots go in blocks of 32; with n = ceil(head_dim / 32) (missing values have code 0) a block holds
  128 n words of key codes    [token][4 n]: word w of a token holds values 8 w .. 8 w + 7
  128 n words of value codes  [piece][g = 0..3][m = 0..15][e]: the word of dimension d = 16 (piece E + e) + m
                              holds tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3 (E = 4 for even n, else 2)
  32 words of key scales, 32 words of value scales
and in a word of eight codes, code j takes four bits from bit 2 + 4 (j // 2) + 16 (j % 2) on, bit 32 being bit 0 again.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "llm_quantization-kernel_amd")

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
#: The largest listed cases: cached values of a decode pass, scores of a prompt pass (padded), appended values.
MOST_CACHED = 48 * 4096 * 8 * 128
MOST_SCORES = 32 * 8192 * 8192
MOST_NEW = 8192 * 32 * 128


# ----------------------------------------------------------------------------- cases

def listed():
    return [
        # a chat's first token after a short question, Llama-2-7B heads: the smallest call
        dict(name="decode_b1_77", kind="decode", b=1, t=1, hq=32, hkv=32, d=128, lmin=77, lmax=77, idle=0, page=64,
             dtype="fp16"),
        # one user, a very long document, grouped heads
        dict(name="decode_b1_131071_gqa", kind="decode", b=1, t=1, hq=32, hkv=8, d=128, lmin=131071, lmax=131071,
             idle=0, page=128, dtype="bf16"),
        # a serving batch of Llama-2-7B at its full context, requests of every age and an idle slot
        dict(name="decode_b32_4096", kind="decode", b=32, t=1, hq=32, hkv=32, d=128, lmin=64, lmax=4096, idle=1,
             page=64, dtype="fp16"),
        # the largest serving batch, grouped heads, long contexts
        dict(name="decode_b64_8192_gqa", kind="decode", b=64, t=1, hq=32, hkv=8, d=128, lmin=1024, lmax=8192, idle=0,
             page=128, dtype="bf16"),
        # four drafted tokens of each request checked at once
        dict(name="decode_b8_t4_gqa", kind="decode", b=8, t=4, hq=32, hkv=8, d=128, lmin=500, lmax=2049, idle=0,
             page=32, dtype="fp16"),
        # OPT-2.7B's heads of 80 in a model loaded in full precision
        dict(name="decode_b5_d80_fp32", kind="decode", b=5, t=1, hq=32, hkv=32, d=80, lmin=200, lmax=1501, idle=0,
             page=64, dtype="fp32"),
        # one decode step's new tokens of a serving batch
        dict(name="append_b64", kind="append", b=64, hkv=8, d=128, smin=100, smax=4000, nmin=1, nmax=1, page=64,
             dtype="bf16"),
        # packed prompts entering the cache, some behind a prefix
        dict(name="append_prompts", kind="append", b=6, hkv=32, d=128, smin=1, smax=300, nmin=200, nmax=1999, page=64,
             dtype="fp16"),
        # a short question
        dict(name="prompt_77", kind="prompt", b=1, hq=32, hkv=32, d=128, lmin=77, lmax=77, dtype="fp16"),
        # prompts of several requests in one pass, grouped heads
        dict(name="prompt_packed_gqa", kind="prompt", b=9, hq=32, hkv=8, d=128, lmin=16, lmax=2047, dtype="bf16"),
        # a long document, grouped heads
        dict(name="prompt_8192_gqa", kind="prompt", b=1, hq=32, hkv=8, d=128, lmin=8192, lmax=8192, dtype="bf16"),
        # OPT-2.7B's heads of 80, its full context
        dict(name="prompt_d80", kind="prompt", b=4, hq=32, hkv=32, d=80, lmin=1500, lmax=2048, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "decode", "decode", "append"])
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    d = rng.choice([64, 80, 96, 128, 128, 128, 256])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    hkv = rng.choice([1, 2, 4, 8, 8, 16, 32]) if group == 1 else rng.choice([1, 2, 4, 8])
    page = rng.choice([32, 64, 64, 128, 256])
    if kind == "prompt":
        b = _log_int(rng, 1, 16)
        most = MOST_SCORES // (64 if dtype == "fp32" else 1)
        lmax = _log_int(rng, 1, max(1, int(math.sqrt(most / (b * hkv * group)))))
        lmax = min(lmax, 8192)
        return dict(kind=kind, b=b, hq=hkv * group, hkv=hkv, d=d, lmin=max(1, lmax // rng.choice([1, 4, 64])), lmax=lmax,
                    dtype=dtype)
    if kind == "decode":
        b = _log_int(rng, 1, 64)
        t = rng.choice([1, 1, 1, 2, 4, 7])
        lmax = _log_int(rng, max(16, t), min(131072, MOST_CACHED // (b * hkv * d)))
        return dict(kind=kind, b=b, t=t, hq=hkv * group, hkv=hkv, d=d, lmin=max(t, lmax // rng.choice([1, 4, 64])),
                    lmax=lmax, idle=rng.choice([0, 0, 1]) if b > 1 else 0, page=page, dtype=dtype)
    if rng.random() < 0.5:
        b, nmin, nmax = _log_int(rng, 1, 256), 1, 1
    else:
        b = _log_int(rng, 1, 16)
        nmax = _log_int(rng, 1, max(1, min(8192, MOST_NEW // (b * hkv * d))))
        nmin = max(1, nmax // rng.choice([1, 4, 64]))
    return dict(kind=kind, b=b, hkv=hkv, d=d, smin=1, smax=_log_int(rng, 1, 4096), nmin=nmin, nmax=nmax, page=page,
                dtype=dtype)


def _lengths(case, lo, hi, salt):
    """A length of each sequence, spread over the logarithm of its range; the longest first."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")) + salt)
    return [hi] + [_log_int(rng, lo, hi) for _ in range(case["b"] - 1)]


def _decode_lengths(case):
    n = _lengths(case, case["lmin"], case["lmax"], "cached")
    return n[:len(n) - case["idle"]] + [0] * case["idle"]


# ----------------------------------------------------------------------------- inputs

def _gen(seed, what):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + what) & 0x7FFFFFFFFFFF)


def _vectors(seed, what, rows, heads, d, dtype):
    """Keys or values: normal, with the few large channels that a language model's have."""
    g = _gen(seed, what)
    x = torch.randn(rows, heads, d, generator=g, device="cuda")
    x *= torch.where(torch.rand(heads, d, generator=g, device="cuda") < 1 / 64, 4.0, 1.0)
    return x.to(dtype)


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(seed, lengths, page):
    """(table [sequences, most pages], pages in the pool): each sequence's pages anywhere in the pool, -1 behind
    its last."""
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + 3
    ids = torch.randperm(pool, generator=_gen(seed, 50), device="cuda").int()
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = _starts(need)
    for i, n in enumerate(need):
        table[i, :n] = ids[at[i]:at[i + 1]]
    return table, pool


def _words(d):
    """(n, words of a block) for heads of d values."""
    n = -(-d // 32)
    return n, 256 * n + 64


def _pool(seed, what, pool, heads, page, d):
    """Codes [pool, heads, page, d], and words of scale and zero point [pool, heads, page], of keys or values."""
    g = _gen(seed, what)
    c = torch.randn(pool, heads, page, d, generator=g, device="cuda").mul_(2.5).add_(7.5).round_().clamp_(0, 15)
    s = torch.rand(pool, heads, page, generator=g, device="cuda") * 0.2 + 0.3
    z = torch.randint(6, 10, (pool, heads, page), generator=g, device="cuda", dtype=torch.int32)
    return c.to(torch.uint8), (s.view(torch.int32) & ~15) | z


def _shifts(device):
    j = torch.arange(8, device=device, dtype=torch.int32)
    return 4 * (j // 2) + 16 * (j % 2)


def _turned(w):
    """Words two bits to the left, the top two at the bottom."""
    return (w << 2) | ((w >> 30) & 3)


def _join(c):
    """Eight codes along the last axis -> one word."""
    return _turned((c.to(torch.int32) << _shifts(c.device)).sum(-1, dtype=torch.int32))


def _split(w):
    w = ((w >> 2) & 0x3FFFFFFF) | (w << 30)
    return (w[..., None] >> _shifts(w.device)) & 15


def _one(w, shift):
    """The code of each word that lies `shift` + 2 bits up."""
    return ((((w >> 2) & 0x3FFFFFFF) | (w << 30)) >> shift) & 15


def _pages_of(kc, kw, vc, vw):
    """The pool's words from codes [pool, heads, page, d] and scale words [pool, heads, page]."""
    pool, heads, page, d = kc.shape
    n, size = _words(d)
    e, blocks = 4 if n % 2 == 0 else 2, page // 32
    if d != 32 * n:
        kc, vc = (torch.nn.functional.pad(c, (0, 32 * n - d)) for c in (kc, vc))
    out = torch.empty(pool, heads, blocks, size, dtype=torch.int32, device=kc.device)
    out[..., :128 * n] = _join(kc.view(pool, heads, blocks, 128 * n, 8))
    v = vc.view(pool, heads, blocks, 2, 4, 4, 2 * n // e, e, 16)      # token = 16 hi + 4 g + lo, d = (piece, e, m)
    v = v.permute(0, 1, 2, 6, 4, 8, 7, 3, 5)                           # piece, g, m, e, hi, lo
    out[..., 128 * n:256 * n] = _join(v.reshape(pool, heads, blocks, 128 * n, 8))
    out[..., 256 * n:256 * n + 32] = kw.view(pool, heads, blocks, 32)
    out[..., 256 * n + 32:] = vw.view(pool, heads, blocks, 32)
    return out.view(pool, heads, blocks * size)


def prepare(case, seed):
    kind, dtype, d, hkv = case["kind"], DTYPES[case["dtype"]], case["d"], case["hkv"]
    st = {"kind": kind, "d": d, "dtype": dtype}
    if kind == "prompt":
        n = _lengths(case, case["lmin"], case["lmax"], "prompt")
        rows = sum(n)
        st.update(q=_vectors(seed, 0, rows, case["hq"], d, dtype), k=_vectors(seed, 1, rows, hkv, d, dtype),
                  v=_vectors(seed, 2, rows, hkv, d, dtype), cu=_int32(_starts(n)), longest=max(n))
        return st
    page = case["page"]
    st["page"] = page
    if kind == "decode":
        n = _decode_lengths(case)
        st["table"], pool = _table(seed, n, page)
        st["pages"] = _pages_of(*_pool(seed, 1, pool, hkv, page, d), *_pool(seed, 2, pool, hkv, page, d))
        st["lens"] = _int32(n)
        st["q"] = _vectors(seed, 0, case["b"] * case["t"], case["hq"], d, dtype).view(case["b"], case["t"], case["hq"], d)
        return st
    held = _lengths(case, case["smin"], case["smax"], "held")
    new = _lengths(case, case["nmin"], case["nmax"], "new")
    rows = sum(new)
    st["table"], pool = _table(seed, [h + m for h, m in zip(held, new)], page)
    st["pages"] = _pages_of(*_pool(seed, 3, pool, hkv, page, d), *_pool(seed, 4, pool, hkv, page, d))
    st.update(lens=_int32([h + m for h, m in zip(held, new)]), cu=_int32(_starts(new)), rows=rows,
              k=_vectors(seed, 1, rows, hkv, d, dtype), v=_vectors(seed, 2, rows, hkv, d, dtype))
    return st


# ----------------------------------------------------------------------------- passes

def run(st):
    if own:
        return _own(st)
    return {"prompt": _prompt, "decode": _decode, "append": _append}[st["kind"]](st)


def _own(st):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import crispybits_kernels as ck
    if st["kind"] == "prompt":
        return ck.prompt_attention(st["q"], st["k"], st["v"], st["cu"], st["longest"])
    cache = ck.KV4Cache(st["pages"], st["page"], st["d"])
    if st["kind"] == "decode":
        return ck.kv4_attention(st["q"], cache, st["table"], st["lens"])
    ck.kv4_append(cache, st["k"], st["v"], st["table"], st["lens"], st["cu"])
    return ck.kv4_read(cache, st["table"], st["lens"], st["cu"], st["rows"], st["dtype"])


def _softmax_times(s, seen, v):
    """softmax(s) v over the last axis of s where ``seen``; rows that see nothing give zeros."""
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _padded(cu, longest):
    """Rows of the packed tensor [sequences, longest] and whether each is one of the sequence's."""
    at = torch.arange(longest, device=cu.device)
    real = at < (cu[1:] - cu[:-1])[:, None]
    return (cu[:-1, None] + at).clamp_max(int(1e9)).where(real, cu[:-1, None].clamp_max(0)).long(), real


def _prompt(st):
    q, k, v = st["q"], st["k"], st["v"]
    heads, d = q.shape[1:]
    hkv = k.shape[1]
    rows, real = _padded(st["cu"], st["longest"])
    b, n = rows.shape
    q, k, v = (x.float()[rows].permute(0, 2, 1, 3) for x in (q, k, v))                     # [b, heads, n, d]
    k, v = (x.where(real[:, None, :, None], 0).contiguous() for x in (k, v))
    q = (q * d ** -0.5).reshape(b, hkv, heads // hkv * n, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(b, hkv, heads // hkv, n, n)
    at = torch.arange(n, device=q.device)
    seen = at[None, :] <= at[:, None]
    s = _softmax_times(s, seen, v[:, :, None])
    return s.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d)[real].to(st["dtype"])


def _unpack(pages, d):
    """Pages [..., words] -> key codes, value codes [..., page, d] and scale words [..., page] of each."""
    n, size = _words(d)
    e = 4 if n % 2 == 0 else 2
    lead = pages.shape[:-1]
    w = pages.reshape(*lead, -1, size)
    blocks = w.shape[-2]
    k = _split(w[..., :128 * n]).reshape(*lead, blocks * 32, 32 * n)[..., :d]
    v = _split(w[..., 128 * n:256 * n]).reshape(-1, 2 * n // e, 4, 16, e, 2, 4)            # piece, g, m, e, hi, lo
    v = v.permute(0, 5, 2, 6, 1, 4, 3).reshape(*lead, blocks * 32, 32 * n)[..., :d]
    return (k, w[..., 256 * n:256 * n + 32].reshape(*lead, -1), v, w[..., 256 * n + 32:].reshape(*lead, -1))


def _value(c, word):
    s = word.view(torch.float32)[..., None]
    return s * (c - (word & 15)[..., None]).float()


def _decode(st):
    q, table, lens, d = st["q"], st["table"], st["lens"], st["d"]
    b, t, heads, _ = q.shape
    pages = st["pages"][table.clamp_min(0)]                                                # [b, pages, hkv, words]
    hkv = pages.shape[2]
    kc, kw, vc, vw = _unpack(pages.transpose(1, 2), d)
    n = table.shape[1] * st["page"]
    at = torch.arange(n, device=q.device)
    k, v = (_value(c, w.contiguous()).reshape(b, hkv, n, d).where((at < lens[:, None])[:, None, :, None], 0)
            for c, w in ((kc, kw), (vc, vw)))
    qs = (q.float() * d ** -0.5).view(b, t, hkv, heads // hkv, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    s = torch.matmul(qs, k.transpose(-1, -2).contiguous()).view(b, hkv, t, heads // hkv, n)
    last = lens[:, None] - t + torch.arange(t, device=q.device)                            # [b, t]
    seen = at <= last[..., None]                                                           # [b, t, n]
    o = _softmax_times(s, seen[:, None, :, None], v[:, :, None])
    return o.permute(0, 2, 1, 3, 4).reshape(b, t, heads, d).to(st["dtype"])


def _quantize(x):
    """Codes int32 and scale words of vectors x [..., d]; in 64 bits, since a border moves whole codes."""
    x = x.double()
    lo, hi = x.amin(-1).clamp_max(0), x.amax(-1).clamp_min(0)
    z = torch.round(-15 * lo / (hi - lo).clamp_min(1e-300)).int()
    word = (((hi - lo) / 15).float().clamp_min(2.0 ** -100).view(torch.int32) & ~15) | z
    s = word.view(torch.float32).double()[..., None]
    return (torch.round(x / s) + z[..., None]).clamp(0, 15).int(), word


def _slots(st):
    """Page and slot of each new token."""
    cu, lens = st["cu"].long(), st["lens"].long()
    row = torch.arange(st["rows"], device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    at = lens[seq] - (cu[seq + 1] - cu[seq]) + row - cu[seq]
    return st["table"].long()[seq, at // st["page"]], at % st["page"]


def _append(st):
    d, page = st["d"], st["page"]
    n, size = _words(d)
    e = 4 if n % 2 == 0 else 2
    heads = st["k"].shape[1]
    w = st["pages"].view(st["pages"].shape[0], heads, page // 32, size)
    pg, slot = _slots(st)
    blk, tok = slot // 32, slot % 32
    (kc, kw), (vc, vw) = _quantize(st["k"]), _quantize(st["v"])
    if d != 32 * n:
        kc = torch.nn.functional.pad(kc, (0, 32 * n - d))
    h = torch.arange(heads, device=pg.device)
    pg, blk, tok = pg[:, None], blk[:, None], tok[:, None]
    w[pg, h, blk, 256 * n + tok] = kw
    w[pg, h, blk, 256 * n + 32 + tok] = vw
    at = torch.arange(4 * n, device=pg.device)
    w[pg[..., None], h[:, None], blk[..., None], tok[..., None] * (4 * n) + at] = _join(kc.view(-1, heads, 4 * n, 8))
    # a value's word is shared with seven other tokens: add what its code changes by
    dd = torch.arange(d, device=pg.device)
    tile, m = dd // 16, dd % 16
    g, j = tok % 16 // 4, tok % 4 + 4 * (tok // 16)
    at = 128 * n + ((tile // e) * 64 + g[..., None] * 16 + m) * e + tile % e                # [rows, 1, d]
    sh = (4 * (j // 2) + 16 * (j % 2))[..., None].int()
    idx = (pg[..., None], h[:, None], blk[..., None], at)
    old = _one(w[idx], sh)
    w.index_put_(idx, _turned(vc << sh) - _turned(old << sh), accumulate=True)
    # and the tokens' values back
    k = _split(w[pg[..., None], h[:, None], blk[..., None], tok[..., None] * (4 * n) + torch.arange(4 * n, device=pg.device)])
    v = _one(w[idx], sh)
    return (_value(k.reshape(-1, heads, 32 * n)[..., :d], w[pg, h, blk, 256 * n + tok]).to(st["dtype"]),
            _value(v, w[pg, h, blk, 256 * n + 32 + tok]).to(st["dtype"]))


# ----------------------------------------------------------------------------- what a pass needs

def work(case):
    kind, d, hkv, e = case["kind"], case["d"], case["hkv"], ESIZE[case["dtype"]]
    if kind == "prompt":
        n = _lengths(case, case["lmin"], case["lmax"], "prompt")
        return {"bytes": sum(n) * d * e * 2 * (case["hq"] + hkv) + 4 * (len(n) + 1),
                "flops": 2 * d * case["hq"] * sum(m * (m + 1) for m in n)}
    if kind == "decode":
        n, t = _decode_lengths(case), case["t"]
        seen = sum(max(0, m - t + 1 + i) for m in n for i in range(t))
        return {"bytes": sum(n) * hkv * (d + 8) + 2 * case["b"] * t * case["hq"] * d * e
                + 4 * sum(1 + -(-m // case["page"]) for m in n), "flops": 4 * d * case["hq"] * seen}
    rows = sum(_lengths(case, case["nmin"], case["nmax"], "new"))
    return {"bytes": rows * hkv * (4 * d * e + 2 * (d + 8)), "flops": rows * hkv * d * 2 * 8}


# ----------------------------------------------------------------------------- in 64 bits

def _exact_rows(q, k, v, first):
    """Attention of q [t, heads, d], row i of which sees keys 0 .. first + i of k, v [n, hkv, d]: row by head."""
    t, heads, d = q.shape
    n, hkv, _ = k.shape
    out = torch.empty(t, heads, d, dtype=torch.float64, device=q.device)
    seen = torch.arange(n, device=q.device)[None, :] <= first + torch.arange(t, device=q.device)[:, None]
    for h in range(heads):
        s = (q[:, h] @ k[:, h // (heads // hkv)].T / math.sqrt(d)).masked_fill(~seen, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, h // (heads // hkv)]
    return torch.where(seen.any(-1)[:, None, None], out, 0.0)


def _value64(c, word):
    return word.view(torch.float32).double()[..., None] * (c.double() - (word & 15).double()[..., None])


def _quantized64(x):
    """The values that x [rows, heads, d] is held as: 15 steps over a range that holds zero, the scale a float
    word whose low four bits are the zero point, each value at the nearest step (halves to the even one)."""
    x = x.double()
    low, high = torch.minimum(x.amin(-1), x.new_zeros(())), torch.maximum(x.amax(-1), x.new_zeros(()))
    span = high - low
    zero = torch.where(span > 0, torch.round(-15 * low / span), 0.0)
    scale = torch.maximum((span / 15).float(), torch.tensor(2.0 ** -100, device=x.device))
    scale = ((scale.view(torch.int32) // 16) * 16 + zero.int()).view(torch.float32).double()
    code = torch.round(x / scale[..., None]) + zero[..., None]
    return scale[..., None] * (code.clamp(0, 15) - zero[..., None])


def exact(case, seed):
    kind, dtype, d, hkv = case["kind"], DTYPES[case["dtype"]], case["d"], case["hkv"]
    if kind == "prompt":
        n = _lengths(case, case["lmin"], case["lmax"], "prompt")
        at = _starts(n)
        q, k, v = (_vectors(seed, i, at[-1], h, d, dtype).double() for i, h in enumerate((case["hq"], hkv, hkv)))
        return torch.cat([_exact_rows(q[a:z], k[a:z], v[a:z], 0) for a, z in zip(at, at[1:])])
    if kind == "decode":
        n, b, t = _decode_lengths(case), case["b"], case["t"]
        table, pool = _table(seed, n, case["page"])
        q = _vectors(seed, 0, b * t, case["hq"], d, dtype).double().view(b, t, case["hq"], d)
        held = [_pool(seed, what, pool, hkv, case["page"], d) for what in (1, 2)]
        out = torch.zeros(b, t, case["hq"], d, dtype=torch.float64, device="cuda")
        for i, m in enumerate(n):
            if m:
                ids = table[i, :-(-m // case["page"])].long()
                k, v = (_value64(c[ids], w[ids]).transpose(1, 2).reshape(-1, hkv, d)[:m] for c, w in held)
                out[i] = _exact_rows(q[i], k, v, m - t)
        return out
    rows = sum(_lengths(case, case["nmin"], case["nmax"], "new"))
    return tuple(_quantized64(_vectors(seed, what, rows, hkv, d, dtype)) for what in (1, 2))
