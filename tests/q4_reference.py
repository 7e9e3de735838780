"""The 4-bit cache's rows and the attention over them by their definitions, in 64 bits on the host (numpy)."""
import numpy as np

S, ROW = 128, 80


def quantise(x):
    """x float64 [..., 128] -> int8 [..., 80].  Codes by comparison with the middles between levels, even codes where they are met"""
    x = np.asarray(x, np.float64)
    g = x.reshape(x.shape[:-1] + (4, 32))
    spoilt = ~(np.abs(x) <= 65024).all(-1)
    g = np.where(spoilt[..., None, None], 0.0, g)
    most = np.abs(g).max(-1, keepdims=True)
    u = np.full_like(most, 2.0 ** -24)
    while (most > 2032 * u).any():
        u = np.where(most > 2032 * u, 2 * u, u)
    t = g / u
    lo, hi = np.rint(t.min(-1, keepdims=True)) + 0.0, np.rint(t.max(-1, keepdims=True))
    s = np.ceil((hi - lo) / 15) + 0.0  # (zeros are positive)
    code = np.zeros(t.shape, np.int64)
    for j in range(15):
        middle = lo + (j + 0.5) * s
        code += ((t > middle) | ((t == middle) & (j % 2 == 1))) & (s > 0)
    d, m = (s * u).astype(np.float16), (lo * u).astype(np.float16)
    m[spoilt] = np.nan
    words = code.reshape(code.shape[:-2] + (16, 8)).astype(np.uint64)
    i = np.arange(8)
    words = (words << (4 * (i // 2) + 16 * (i % 2)).astype(np.uint64)).sum(-1).astype(np.uint32)
    pairs = np.concatenate((d, m), axis=-1)
    return np.concatenate((words.view(np.int8).reshape(x.shape[:-1] + (64,)), np.ascontiguousarray(pairs).view(np.int8).reshape(x.shape[:-1] + (16,))), axis=-1)


def values(rows):
    """int8 [..., 80] -> float64 [..., 128]"""
    rows = np.ascontiguousarray(rows)
    words, pairs = rows[..., :64].copy().view(np.uint32), rows[..., 64:].copy().view(np.float16).astype(np.float64)
    i = np.arange(8, dtype=np.uint32)
    code = (words[..., None] >> (4 * (i // 2) + 16 * (i % 2)).astype(np.uint32)) & np.uint32(15)
    code = code.reshape(rows.shape[:-1] + (4, 32)).astype(np.float64)
    return (code * pairs[..., 0::2, None] + pairs[..., 1::2, None]).reshape(rows.shape[:-1] + (S,))


def turned(x, inv_freq, pos):
    """x float64 [..., 128], pos [...]: pairs (i, i + half)"""
    half = len(inv_freq)
    a = np.asarray(pos, np.float64)[..., None] * np.asarray(inv_freq, np.float64)
    lo, hi = x[..., :half], x[..., half:2 * half]
    return np.concatenate((lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a), x[..., 2 * half:]), axis=-1)


def extents(lengths, q_lens, qL, maxlen):
    out = []
    for b in range(len(lengths)):
        n = min(max(int(lengths[b]), 0), maxlen)
        t = qL if q_lens is None else min(max(int(q_lens[b]), 0), qL)
        out.append((n, min(t, maxlen - n)))
    return out


def write(cache, k, v, layer, lengths, q_lens, inv_freq):
    """cache int8 [planes,B,Hkv,maxlen,80], in place; k, v [B,L,Hkv,128]"""
    B, L = k.shape[:2]
    for b, (n, t) in enumerate(extents(lengths, q_lens, L, cache.shape[3])):
        new = np.asarray(k[b, :t], np.float64)
        if inv_freq is not None:
            new = turned(new, inv_freq, np.broadcast_to(n + np.arange(t)[:, None], new.shape[:-1]))
        cache[2 * layer, b, :, n:n + t] = quantise(new).transpose(1, 0, 2)
        cache[2 * layer + 1, b, :, n:n + t] = quantise(v[b, :t]).transpose(1, 0, 2)


def attention(q, cache, layer, lengths, q_lens, inv_freq):
    """over a cache that holds the new rows: (out float64 [B,L,H,128], what an fp32 evaluation by halves may be off by [B,L,H]).

    The error, with e = 2^-24: a query's rotation in fp32 2 e of each value and its two halves 4 e of its largest; 8 + 2 sums of a score each
    off by e of the absolute products; the score in units of log2 by 3 e of itself.  Such an error x in a score changes weights by a part x, the result by 2 x max|V|.  The
    weights: exp2 and two halves 4 e, 2^-28 of the largest in all; sums of them over rows / 128 + 10 steps and the division each e, twice (weights, products)."""
    B, L, H, _ = q.shape
    Hkv, maxlen = cache.shape[2:4]
    g = H // Hkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape[:-1])
    e = 2.0 ** -24
    for b, (n, t) in enumerate(extents(lengths, q_lens, L, maxlen)):
        K, V = values(cache[2 * layer, b, :, :n + t]), values(cache[2 * layer + 1, b, :, :n + t])
        for l in range(t):
            rows = n + l + 1
            x = turned(np.asarray(q[b, l], np.float64), inv_freq, np.full(H, n + l)).reshape(Hkv, g, S)
            s = np.einsum("hgd,hrd->hgr", x, K[:, :rows]) / np.sqrt(S)
            w = np.exp(s - s.max(-1, keepdims=True))
            out[b, l] = (np.einsum("hgr,hrd->hgd", w, V[:, :rows]) / w.sum(-1, keepdims=True)).reshape(H, S)
            size = np.abs(K[:, :rows])
            products = np.einsum("hgd,hrd->hgr", np.abs(x), size).max(-1)
            largest = np.abs(x).max(-1) * size.sum(-1).max(-1)[:, None]
            score = (12 * products + 4 * largest) * e / np.sqrt(S) + 3 * e * np.abs(s).max(-1)
            top = np.abs(V[:, :rows]).max((-1, -2))[:, None]
            tol[b, l] = (top * (2 * score + (4 + 16 + 2 * (rows / 128 + 12)) * e + rows * 2.0 ** -28) + 2.0 ** -36).reshape(H)
    return out, tol
