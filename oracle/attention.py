"""CPU oracle of the attention ops, in float64: the 4-bit cache's format word by word, its append and read,
attention over it, and causal attention over packed prompts.

The functions without a leading underscore have the signatures of ``crispybits_kernels._C``, so that the module
serves as its attention backend in CPU tests.  Written from the definitions; shares no code with the product.
"""
import numpy as np
import torch

BLOCK = 32


def _f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _i64(t):
    return t.detach().cpu().to(torch.int64).numpy()


def kv4_page_words(head_dim, page_size):
    if head_dim <= 0 or head_dim > 256 or head_dim % 8:
        raise RuntimeError("head_dim must be a multiple of 8 up to 256")
    if page_size < 32 or page_size > 65536 or page_size & (page_size - 1):
        raise RuntimeError("page_size must be a power of two from 32 to 65536")
    return page_size // BLOCK * _block_words(head_dim)


def _ns(d):
    return -(-d // 32)


def _block_words(d):
    return 256 * _ns(d) + 64


def quantize(x):
    """Codes (int64) and scale words (uint32) of vectors x [..., D] (float64 values of the input's type)."""
    fine = np.isfinite(x).all(-1)
    x = np.where(fine[..., None], x, 0.0)
    lo, hi = np.minimum(x.min(-1), 0.0), np.maximum(x.max(-1), 0.0)
    r = hi - lo
    z = np.where(r > 0, np.rint(-15.0 * lo / np.where(r > 0, r, 1.0)), 0.0).astype(np.int64)
    step = np.maximum((r / 15.0).astype(np.float32), np.float32(2.0 ** -100))
    word = (step.view(np.uint32) & np.uint32(0xFFFFFFF0)) | z.astype(np.uint32)
    s = word.view(np.float32).astype(np.float64)
    c = np.clip(np.rint(x / s[..., None]) + z[..., None], 0, 15).astype(np.int64)
    word = np.where(fine, word, np.uint32(0x7FC00000))
    return np.where(fine[..., None], c, 0), word.astype(np.uint32)


def values(c, word):
    """What codes [..., D] and scale words [...] stand for, as the float32 product."""
    s = word.view(np.float32)
    z = (word & 15).astype(np.int64)
    with np.errstate(invalid="ignore"):
        return s[..., None] * (c - z[..., None]).astype(np.float32)


def _bit(j):
    """First of the four bits of value j of a word; bit 32 is bit 0 again."""
    return 2 + 4 * (j // 2) + 16 * (j % 2)


def _put(word, bit, code):
    """`word` with the code at `bit` replaced."""
    at = lambda v: ((v << bit) | (v << bit >> 32)) & 0xFFFFFFFF     # noqa: E731
    return np.uint32(int(word) & ~at(15) | at(code))


def _get(words, bits):
    w = words.astype(np.uint64)
    return ((w | w << np.uint64(32)) >> np.asarray(bits, dtype=np.uint64) & np.uint64(15)).astype(np.int64)


def k_place(d, t, i):
    """Word (within a block) and bit of value i of token t's key."""
    return t * 4 * _ns(d) + i // 8, _bit(i % 8)


def v_place(d, t, i):
    """Word (within a block) and bit of value i of token t's value vector."""
    ns = _ns(d)
    pw = 4 if ns % 2 == 0 else 2
    tile, m = i // 16, i % 16
    g, j = (t % 16) // 4, t % 4 + 4 * (t // 16)
    return 128 * ns + ((tile // pw * 4 + g) * 16 + m) * pw + tile % pw, _bit(j)


def _slot(table, page_size, num_pages, b, pos):
    """(page, block of the page, token of the block), or None where there is no page."""
    if pos < 0 or pos // page_size >= table.shape[1]:
        return None
    page = table[b, pos // page_size]
    if not 0 <= page < num_pages:
        return None
    return page, pos % page_size // BLOCK, pos % BLOCK


def _rows(lens, cu, rows):
    """(sequence, position) of each packed row; None for rows of no sequence."""
    out = [None] * rows
    if cu is None:
        return [(b, lens[b] - 1) for b in range(len(lens))]
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            out[cu[b] + i] = (b, lens[b] - n + i)
    return out


def kv4_append(pages, page_size, head_dim, k, v, table, lens, cu=None):
    P = pages.numpy().view(np.uint32)
    w = P.reshape(P.shape[0], P.shape[1], -1, _block_words(head_dim))
    tb, ln = _i64(table), _i64(lens)
    (kc, kw), (vc, vw) = quantize(_f64(k)), quantize(_f64(v))
    ns = _ns(head_dim)
    for r, at in enumerate(_rows(ln, None if cu is None else _i64(cu), k.shape[0])):
        slot = at and _slot(tb, page_size, P.shape[0], *at)
        if not slot:
            continue
        page, blk, t = slot
        for h in range(P.shape[1]):
            B = w[page, h, blk]
            B[t * 4 * ns:(t + 1) * 4 * ns] = 0
            for i in range(32 * ns):
                ck, cv = (int(kc[r, h, i]), int(vc[r, h, i])) if i < head_dim else (0, 0)
                x, bit = k_place(head_dim, t, i)
                B[x] = _put(B[x], bit, ck)
                x, bit = v_place(head_dim, t, i)
                B[x] = _put(B[x], bit, cv)
            B[256 * ns + t] = kw[r, h]
            B[256 * ns + 32 + t] = vw[r, h]


def stored(pages, page_size, head_dim, table, b, n):
    """Keys and values [n, heads, D] (float32 values) of positions 0 .. n - 1 of sequence b, and which exist."""
    P = pages.detach().cpu().numpy().view(np.uint32)
    heads, ns = P.shape[1], _ns(head_dim)
    w = P.reshape(P.shape[0], heads, -1, _block_words(head_dim))
    tb = _i64(table)
    k, v = (np.zeros((n, heads, head_dim), np.float32) for _ in range(2))
    there = np.zeros(n, bool)
    i = np.arange(head_dim)
    for pos in range(n):
        slot = _slot(tb, page_size, P.shape[0], b, pos)
        if not slot:
            continue
        page, blk, t = slot
        there[pos] = True
        B = w[page, :, blk]
        for out, place, meta in ((k, k_place, 256 * ns), (v, v_place, 256 * ns + 32)):
            x, bit = place(head_dim, t, i)
            c = _get(B[:, x], np.broadcast_to(bit, i.shape))
            out[pos] = values(c, np.ascontiguousarray(B[:, meta + t]))
    return k, v, there


def kv4_read(pages, page_size, head_dim, table, lens, cu, rows, dtype):
    ln = _i64(lens)
    k, v = (torch.zeros(rows, pages.shape[1], head_dim, dtype=torch.float32) for _ in range(2))
    held = {}
    for r, at in enumerate(_rows(ln, None if cu is None else _i64(cu), rows)):
        if at is None or at[1] < 0:
            continue
        b, pos = at
        if b not in held:
            held[b] = stored(pages, page_size, head_dim, table, b, int(ln[b]))
        k[r], v[r] = torch.from_numpy(held[b][0][pos]), torch.from_numpy(held[b][1][pos])
    return k.to(dtype), v.to(dtype)


def softmax_rows(q, k, v, seen, scale):
    """(out, sum p |v|, scores) of q [t, D] over k, v [n, D] where seen [t, n]; rows that see nothing give zeros."""
    keep = seen.any(0)
    k, v, seen = k[keep], v[keep], seen[:, keep]
    out, mag = np.zeros((q.shape[0], v.shape[1])), np.zeros((q.shape[0], v.shape[1]))
    with np.errstate(invalid="ignore", over="ignore"):
        s = scale * (q @ k.T)
        for r in range(q.shape[0]):
            m = seen[r]
            if not m.any():
                continue
            e = np.exp(s[r, m] - s[r, m].max())
            p = e / e.sum()
            out[r], mag[r] = p @ v[m], p @ np.abs(v[m])
    return out, mag


def attention64(q, pages, page_size, head_dim, table, lens, scale):
    """(out, sum p |v|) float64 [seqs, t, heads, D]."""
    q = _f64(q)
    seqs, t, heads, _ = q.shape
    group = heads // pages.shape[1]
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for b, n in enumerate(_i64(lens)):
        n = int(min(n, table.shape[1] * page_size))
        if n <= 0:
            continue
        k, v, there = stored(pages, page_size, head_dim, table, b, n)
        newest = int(_i64(lens)[b]) - t + np.arange(t)
        seen = (np.arange(n)[None] <= newest[:, None]) & there[None]
        for h in range(heads):
            o = softmax_rows(q[b, :, h], k[:, h // group].astype(np.float64), v[:, h // group].astype(np.float64), seen, scale)
            out[b, :, h], mag[b, :, h] = o
    return out, mag


def kv4_attention(q, pages, page_size, head_dim, table, lens, scale, out=None):
    o = torch.from_numpy(attention64(q, pages, page_size, head_dim, table, lens, scale)[0]).to(q.dtype)
    return o if out is None else out.copy_(o)


def prompt64(q, k, v, cu, scale):
    """(out, sum p |v|) float64 [rows, heads, D]."""
    q, k, v, cu = _f64(q), _f64(k), _f64(v), _i64(cu)
    group = q.shape[1] // k.shape[1]
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for a, z in zip(cu, cu[1:]):
        seen = np.tril(np.ones((z - a, z - a), bool))
        for h in range(q.shape[1]):
            out[a:z, h], mag[a:z, h] = softmax_rows(q[a:z, h], k[a:z, h // group], v[a:z, h // group], seen, scale)
    return out, mag


def prompt_attention(q, k, v, cu, max_seqlen, scale, out=None):
    o = torch.from_numpy(prompt64(q, k, v, cu, scale)[0]).to(q.dtype)
    if out is None:
        return o
    z = int(cu[-1])
    out[int(cu[0]):z] = o[int(cu[0]):z]
    return out
