"""attention_rope_q4 against its formula over what the cache holds, in 64 bits on the host (q4_reference.py, where the tolerance is derived)."""
import math

import numpy as np
import pytest
import torch

import llmops
import q4_reference as ref

pytestmark = pytest.mark.gpu


def _inv_freq(half=64):
    return 1.0 / (10000.0 ** (torch.arange(0, 2 * half, 2).float() / (2 * half)))


def _filled(g, planes, B, Hkv, maxlen, scale=1.0):
    """a cache of rows near N(0, 1), made of codes at random (quick)"""
    if scale != 1.0:
        return torch.from_numpy(ref.quantise((torch.randn(planes, B, Hkv, maxlen, 128, generator=g) * scale).numpy()))
    cache = torch.randint(-128, 128, (planes, B, Hkv, maxlen, 80), generator=g, dtype=torch.int8)
    d = (0.2 + 0.2 * torch.rand(planes, B, Hkv, maxlen, 4, generator=g)).mul(256).round() / 256
    m = -(d * torch.randint(6, 10, d.shape, generator=g))
    cache[..., 64:] = torch.stack((d, m), -1).half().flatten(-2).view(torch.int8)
    return cache


def _check(q, k, v, cache, lengths, q_lens, layer=0, half=64, dev=None):
    """q [B,L,H*128] ..., cache on the host; compares out and the cache; returns out"""
    B, L, width = q.shape
    Hkv = cache.shape[2]
    f = _inv_freq(half)
    want = cache.numpy().copy()
    ref.write(want, k.reshape(B, L, Hkv, 128).numpy(), v.reshape(B, L, Hkv, 128).numpy(), layer, lengths, q_lens, f.numpy())
    expect, tol = ref.attention(q.reshape(B, L, -1, 128).numpy(), want, layer, lengths, q_lens, f.numpy())
    dev = cache.cuda() if dev is None else dev
    out = llmops.attention_rope_q4(q.cuda(), k.cuda(), v.cuda(), f.cuda(), dev, lengths.cuda(), layer, q_lens=None if q_lens is None else q_lens.cuda())
    assert np.array_equal(dev.cpu().numpy(), want)
    got = out.cpu().double().numpy().reshape(expect.shape)
    off = np.abs(got - expect).max(-1)
    assert (off <= tol).all(), (off.max(), tol.flat[off.argmax()], (off / np.maximum(tol, 1e-300)).max())
    for b, (n, t) in enumerate(ref.extents(lengths, q_lens, L, cache.shape[3])):
        assert not got[b, t:].any()  # padding
    return out


def _random(g, B, L, H, Hkv):
    return (torch.randn(B, L, w * 128, generator=g) for w in (H, Hkv, Hkv))


@pytest.mark.parametrize("B,L,H,Hkv,maxlen", [
    (1, 1, 1, 1, 1), (1, 1, 32, 32, 2), (2, 1, 32, 32, 200), (3, 1, 8, 2, 1000), (1, 1, 8, 1, 5000), (5, 1, 16, 4, 129), (70, 1, 4, 2, 300), (130, 1, 2, 1, 40),
    (2, 5, 8, 8, 700), (3, 4, 16, 4, 140), (2, 3, 32, 2, 333), (4, 16, 4, 4, 64), (2, 17, 4, 4, 500), (1, 33, 8, 2, 257), (1, 7, 40, 1, 150), (2, 64, 4, 4, 400),
    (1, 300, 4, 1, 500), (3, 130, 2, 2, 131), (1, 257, 3, 3, 1300), (66, 20, 2, 2, 60),
    (2, 1, 4, 4, 1024), (2, 1, 4, 4, 1025), (3, 6, 8, 2, 900), (2, 8, 16, 4, 1024),
    (1, 20, 4, 4, 512), (2, 24, 4, 4, 513), (1, 25, 2, 2, 400), (3, 5, 16, 4, 510)])
def test_against_the_formula(B, L, H, Hkv, maxlen):
    g = torch.Generator().manual_seed(B * L + maxlen)
    q, k, v = _random(g, B, L, H, Hkv)
    cache = _filled(g, 4, B, Hkv, maxlen)
    lengths = torch.randint(0, max(1, maxlen - L + 1), (B,), generator=g, dtype=torch.int32)
    _check(q, k, v, cache, lengths, None, layer=1)
    # lengths and numbers of tokens outside their ranges too
    lengths = torch.randint(-2, maxlen + 3, (B,), generator=g, dtype=torch.int32)
    q_lens = torch.randint(-1, L + 2, (B,), generator=g, dtype=torch.int32)
    _check(q, k, v, cache, lengths, q_lens)


@pytest.mark.parametrize("B,L,H,Hkv,maxlen", [(64, 1, 32, 8, 3000), (130, 1, 8, 8, 1000), (40, 3, 16, 16, 1500), (70, 40, 8, 4, 700), (9, 150, 16, 8, 1200), (33, 20, 8, 8, 2500),
                                              (16, 1, 32, 16, 2048), (17, 1, 16, 16, 2049), (32, 30, 8, 8, 2000), (33, 1, 32, 32, 300), (9, 5, 32, 32, 1500),
                                              (32, 30, 8, 8, 1000), (64, 20, 8, 8, 2000), (33, 8, 32, 8, 1024)])
def test_the_chip_full_of_workgroups(B, L, H, Hkv, maxlen):
    """shares that differ, sequences past 64: against the formula in 64 bits on the device, over what the cache is read back as; tolerance as in q4_reference.py"""
    g = torch.Generator().manual_seed(B)
    q, k, v = (x.cuda() for x in _random(g, B, L, H, Hkv))
    cache = torch.stack([_filled(g, 2, 1, Hkv, maxlen)[:, 0] for _ in range(4)], 1).repeat(1, -(-B // 4), 1, 1, 1)[:, :B].contiguous().cuda()
    lengths = torch.randint(0, maxlen - L + 1, (B,), generator=g, dtype=torch.int32).cuda()
    q_lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32).cuda() if L > 1 else None
    f, e, G = _inv_freq().cuda(), 2.0 ** -24, H // Hkv
    written = cache.clone()
    llmops.cache_write_q4(k, v, written, lengths, 0, inv_freq=f, q_lens=q_lens)
    out = llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0, q_lens=q_lens).reshape(B, L, H, 128)
    assert torch.equal(cache, written)
    full = llmops.cache_read_q4(cache, maxlen)
    for b in range(B):
        n, t = int(lengths[b]), L if q_lens is None else int(q_lens[b])
        assert not out[b, t:].any()
        if not t:
            continue
        K, V = (full[i, b, :, :n + t].double() for i in (0, 1))
        angle = (n + torch.arange(t, device="cuda")).double()[:, None] * f.double()
        lo, hi = q[b, :t].double().reshape(t, H, 128).chunk(2, dim=-1)
        x = torch.cat((lo * angle.cos()[:, None] - hi * angle.sin()[:, None], hi * angle.cos()[:, None] + lo * angle.sin()[:, None]), -1)
        x = x.reshape(t, Hkv, G, 128).permute(1, 0, 2, 3).reshape(Hkv, t * G, 128).contiguous()
        s = torch.matmul(x, K.transpose(1, 2).contiguous()) / math.sqrt(128)
        seen = (torch.arange(n + t, device="cuda") <= n + torch.arange(t, device="cuda")[:, None]).repeat_interleave(G, 0)
        want = torch.matmul(torch.softmax(s.masked_fill(~seen, -math.inf), -1), V)
        products = torch.matmul(x.abs(), K.abs().transpose(1, 2).contiguous()).amax(-1)
        largest = x.abs().amax(-1) * K.abs().sum(-1).amax(-1)[:, None]
        score = (12 * products + 4 * largest) * e / math.sqrt(128) + 3 * e * s.abs().amax(-1)
        rows = n + t
        tol = V.abs().amax((1, 2))[:, None] * (2 * score + (4 + 16 + 2 * (rows / 128 + 12)) * e + rows * 2.0 ** -28) + 2.0 ** -36
        got = out[b, :t].reshape(t, Hkv, G, 128).permute(1, 0, 2, 3).reshape(Hkv, t * G, 128)
        assert ((got - want).abs().amax(-1) <= tol).all(), b


@pytest.mark.parametrize("L", [1, 3, 40])
def test_empty_full_and_almost(L):
    g = torch.Generator().manual_seed(L)
    maxlen = 300
    lengths = torch.tensor([0, 1, 127, 128, 129, 255, 256, 257, maxlen - 1, maxlen, maxlen - L], dtype=torch.int32)
    B = len(lengths)
    q, k, v = _random(g, B, L, 4, 2)
    _check(q, k, v, _filled(g, 2, B, 2, maxlen), lengths, None)
    _check(q, k, v, _filled(g, 2, B, 2, maxlen), lengths, torch.tensor([0, 0, 1, 1, 0, L, L, 0, 1, 1, L], dtype=torch.int32))


@pytest.mark.parametrize("half", [64, 32, 1, 50])
def test_part_of_the_dims_turns(half):
    g = torch.Generator().manual_seed(half)
    q, k, v = _random(g, 2, 3, 4, 2)
    _check(q, k, v, _filled(g, 2, 2, 2, 90), torch.tensor([5, 80], dtype=torch.int32), None, half=half)


def test_columns_of_a_projection():
    g = torch.Generator().manual_seed(3)
    B, L, H, Hkv = 2, 4, 8, 2
    qkv = torch.randn(B, L, (H + 2 * Hkv) * 128, generator=g)
    cache, lengths, f = _filled(g, 2, B, Hkv, 200).cuda(), torch.tensor([100, 7], dtype=torch.int32, device="cuda"), _inv_freq().cuda()
    other = cache.clone()
    x = qkv.cuda()
    keep = x.clone()
    q, k, v = x[..., :H * 128], x[..., H * 128:(H + Hkv) * 128], x[..., (H + Hkv) * 128:]
    a = llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0)
    b = llmops.attention_rope_q4(q.contiguous(), k.contiguous(), v.contiguous(), f, other, lengths, 0)
    assert torch.equal(a, b) and torch.equal(cache, other) and torch.equal(x, keep)


@pytest.mark.parametrize("L,H,Hkv", [(1, 4, 4), (4, 8, 2), (70, 2, 2)])
def test_large_and_small_magnitudes(L, H, Hkv):
    g = torch.Generator().manual_seed(5)
    for scale, q_scale in ((1.0, 30.0), (1000.0, 0.002), (2.0 ** -12, 1000.0), (1.0, 1e-30), (1.0, 1e30)):
        q, k, v = _random(g, 2, L, H, Hkv)
        cache = _filled(g, 2, 2, Hkv, 400, scale)
        if q_scale < 1e20:
            _check(q * q_scale, k * scale, v * scale, cache, torch.tensor([300, 129], dtype=torch.int32), None)
        else:  # one row takes all the weight
            out = llmops.attention_rope_q4((q * q_scale).cuda(), k.cuda(), v.cuda(), _inv_freq().cuda(), cache.cuda(), torch.tensor([300, 129], dtype=torch.int32, device="cuda"), 0)
            assert out.isfinite().all()


def test_what_is_not_seen_has_no_effect():
    # rows past a sequence's own hold anything, NaN among it; so do planes of other layers
    g = torch.Generator().manual_seed(6)
    for L, maxlen in ((1, 700), (5, 200), (80, 300)):
        q, k, v = _random(g, 3, L, 4, 2)
        cache = _filled(g, 4, 3, 2, maxlen)
        lengths = torch.tensor([0, 60, maxlen - L], dtype=torch.int32)
        for b, n in enumerate(lengths.tolist()):
            cache[2:, b, :, n + L:, 64:] = torch.full((8,), math.nan, dtype=torch.float16).view(torch.int8)
            cache[2:, b, :, n:n + L, 64:] = torch.full((8,), math.inf, dtype=torch.float16).view(torch.int8)
        cache[:2, ..., 64:] = torch.full((8,), math.nan, dtype=torch.float16).view(torch.int8)
        _check(q, k, v, cache, lengths, None, layer=1)


@pytest.mark.parametrize("L,G", [(6, 1), (6, 4), (40, 1), (100, 2)])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_nan_reaches_those_who_see_it(L, G, which):
    g = torch.Generator().manual_seed(7)
    Hkv, at, n = 2, 3, 37
    q, k, v = _random(g, 1, L, Hkv * G, Hkv)
    cache, lengths, f = _filled(g, 2, 1, Hkv, 200).cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), _inv_freq().cuda()
    clean = llmops.attention_rope_q4(q.cuda(), k.cuda(), v.cuda(), f, cache.clone(), lengths, 0)
    dict(q=q, k=k, v=v)[which][0, at, 5] = math.nan  # (head 0)
    out = llmops.attention_rope_q4(q.cuda(), k.cuda(), v.cuda(), f, cache, lengths, 0).reshape(L, Hkv, G, 128)
    clean = clean.reshape(L, Hkv, G, 128)
    if which == "q":
        assert out[at, 0, 0].isnan().all()
        clean[at, 0, 0] = out[at, 0, 0] = 0.0
    else:
        assert out[at:, 0].isnan().all()
        clean[at:, 0] = out[at:, 0] = 0.0
    assert torch.equal(out, clean)


def test_same_bits_every_time_whatever_the_capacity_is_filled_with():
    g = torch.Generator().manual_seed(8)
    q, k, v = _random(g, 9, 1, 16, 4)
    cache, lengths, f = _filled(g, 2, 9, 4, 3000), torch.randint(0, 2999, (9,), generator=g, dtype=torch.int32), _inv_freq().cuda()
    a = [llmops.attention_rope_q4(q.cuda(), k.cuda(), v.cuda(), f, cache.cuda(), lengths.cuda(), 0) for _ in range(3)]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])


def test_offsets_past_32_bits():
    heads, maxlen = 60, 1 << 20  # 5 GB a plane
    g = torch.Generator().manual_seed(9)
    cache = torch.zeros(2, 1, heads, maxlen, 80, dtype=torch.int8, device="cuda")
    n = 4000
    part = _filled(g, 2, 1, heads, n).cuda()
    cache[..., :n, :] = part
    q, k, v = (x.cuda() for x in _random(g, 1, 2, heads, heads))
    lengths, f = torch.tensor([n - 2], dtype=torch.int32, device="cuda"), _inv_freq().cuda()
    a = llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0)
    b = llmops.attention_rope_q4(q, k, v, f, part, lengths, 0)
    assert (a - b).abs().max() <= 2e-6 * b.abs().max()  # (other shares: sums in another order, 32 e of |V| here and there)
    assert torch.equal(cache[..., n - 2:n, :], part[..., n - 2:, :])
    lengths.fill_(maxlen - 2)  # 2^20 rows
    out = llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0)
    assert out.isfinite().all()
    assert cache[:, 0, :, -2:].flatten(3).any(-1).all()


def test_one_graph_serves_following_steps():
    g = torch.Generator().manual_seed(10)
    B, H, Hkv, maxlen, f = 3, 8, 2, 500, _inv_freq().cuda()
    for L in (1, 3, 60):
        q, k, v = (x.cuda() for x in _random(g, B, L, H, Hkv))
        start = _filled(g, 2, B, Hkv, maxlen).cuda()
        cache, lengths = start.clone(), torch.zeros(B, dtype=torch.int32, device="cuda")
        q_lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0, q_lens=q_lens)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = llmops.attention_rope_q4(q, k, v, f, cache, lengths, 0, q_lens=q_lens)
        torch.cuda.synchronize()
        for step, lens in enumerate(([0, 1, 2], [300, 5, 440], [128, 127, 129], [499, 500, 0])):
            lengths.copy_(torch.tensor(lens)), q_lens.copy_(torch.tensor([L, step, max(0, L - step)])), cache.copy_(start)
            q.copy_(torch.randn(q.shape, generator=g))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            other = start.clone()
            want = llmops.attention_rope_q4(q, k, v, f, other, lengths, 0, q_lens=q_lens)
            assert torch.equal(out, want) and torch.equal(cache, other)


def test_two_streams_at_once():
    g = torch.Generator().manual_seed(11)
    sets = []
    for _ in range(2):
        q, k, v = (x.cuda() for x in _random(g, 4, 1, 32, 8))
        sets.append((q, k, v, _filled(g, 2, 4, 8, 4000).cuda(), torch.tensor([3000, 17, 2500, 3998], dtype=torch.int32, device="cuda")))
    f = _inv_freq().cuda()
    want = [llmops.attention_rope_q4(q, k, v, f, c.clone(), n, 0) for q, k, v, c, n in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, (q, k, v, c, n), to in zip(streams, sets, got):
            with torch.cuda.stream(s):
                to.append(llmops.attention_rope_q4(q, k, v, f, c, n, 0))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for to, w in zip(got, want) for x in to)


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    cache, lengths = z(2, 2, 4, 8, 80, dtype=torch.int8), z(2, dtype=torch.int32)
    a = dict(q=z(2, 3, 1024), k=z(2, 3, 512), v=z(2, 3, 512), inv_freq=_inv_freq().cuda(), kv_cache=cache, lengths=lengths, layer_id=0)
    llmops.attention_rope_q4(**a)
    for kw in (dict(q=z(2, 3, 1000)), dict(q=z(2, 3, 640)), dict(q=z(1, 3, 1024)), dict(k=z(2, 3, 1024)), dict(v=z(2, 2, 512)), dict(k=z(2, 3, 512).half()),
               dict(kv_cache=cache.half()), dict(kv_cache=cache[..., :68]), dict(kv_cache=cache[:1]), dict(lengths=lengths[:1]), dict(q_lens=lengths[:1]), dict(layer_id=1),
               dict(inv_freq=z(65)), dict(inv_freq=z(0)), dict(q=z(2, 3, 1025)[..., 1:]), dict(q=z(2, 3, 1024).cpu()), dict(kv_cache=cache.cpu())):
        with pytest.raises(RuntimeError):
            llmops.attention_rope_q4(**{**a, **kw})
    with pytest.raises(RuntimeError):  # rows that lie in the cache
        llmops.attention_rope_q4(**{**a, "k": cache.view(torch.float32).flatten().as_strided((2, 3, 512), (512, 0, 1))})


def test_a_capacity_of_two_million_rows():
    """a prompt of a few thousand tokens over a cache of 2^21 rows: as over a small one, bit for bit (work is shared out by the lengths)"""
    g = torch.Generator().manual_seed(12)
    L, H = 4096, 32
    q, k, v = (x.cuda() for x in _random(g, 1, L, H, 1))
    lengths, f = torch.tensor([10], dtype=torch.int32, device="cuda"), _inv_freq().cuda()
    part = _filled(g, 2, 1, 1, L + 10).cuda()
    cache = torch.zeros(2, 1, 1, 1 << 21, 80, dtype=torch.int8, device="cuda")
    cache[..., :L + 10, :] = part
    a, b = (llmops.attention_rope_q4(q, k, v, f, c, lengths, 0) for c in (cache, part))
    assert torch.equal(a, b) and torch.equal(cache[..., :L + 10, :], part) and not cache[..., L + 10:, :].any()
    lengths.fill_((1 << 21) - L)
    out = llmops.attention_rope_q4(q[:, :5], k[:, :5], v[:, :5], f, cache, lengths, 0)
    assert out.isfinite().all()


@pytest.mark.parametrize("B,L,H,Hkv,maxlen", [(40, 1, 4, 4, 100), (40, 1, 4, 4, 3000), (6, 1, 24, 1, 100), (6, 1, 24, 1, 5000), (6, 1, 40, 1, 100), (3, 4, 64, 1, 600)])
def test_weights_near_the_largest_keep_their_bits(B, L, H, Hkv, maxlen):
    """Rows whose scores lie within half a unit (of log2) of each other; out is their weights' ratios to the largest, times 15/16.  Nothing turns, and scores are
    exact.  With e = 2^-24, roots of mean squares: a weight's two halves 1.75 e (a remainder below 2^-10 of it, cut to 11 bits), exp2 of at most one unit 1.15 e, the sum of
    its two products and the product with 1 / sum 0.6 e; the largest one's 0.6, 0.6 and 0.5 e; the factor's 1.5 e of half a unit 0.5 e: 2.5 e in all, and a fifth for the sample.
    (An argument of exp2 that is rounded between 8 and 16 would alone be off by 16 e / sqrt(12) log 2 = 3.2 e, here and at the largest.)"""
    g = torch.Generator().manual_seed(B + H)
    rows, e = 64, 2.0 ** -24
    k, v = torch.zeros(B, rows, Hkv, 128), torch.zeros(B, rows, Hkv, 128)
    k[..., 0] = torch.randint(-15, 16, (B, rows, Hkv), generator=g) / 8
    k[..., 1] = torch.randint(-7, 8, (B, rows, Hkv), generator=g) / 64
    v[:, torch.arange(rows), :, torch.arange(rows)] = 15 / 16
    cache, f = torch.zeros(2, B, Hkv, maxlen, 80, dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda")
    none = torch.zeros(B, dtype=torch.int32, device="cuda")
    llmops.cache_write_q4(k.cuda(), v.cuda(), cache, none, 0, inv_freq=f)
    K, V = llmops.cache_read_q4(cache, rows).double()
    assert torch.equal(V.cpu().float(), v.transpose(1, 2))
    q = torch.zeros(B, L, H, 128)
    q[..., :2] = torch.randint(1024, 2048, (B, L, H, 1), generator=g) / 1024
    first = rows - L
    new = [x[:, first:].flatten(2).cuda() for x in (k, v)]
    out = llmops.attention_rope_q4(q.flatten(2).cuda(), *new, f, cache, none + first, 0).double().unflatten(-1, (Hkv, H // Hkv, 128))
    off = []
    for l in range(L):
        n = first + l + 1
        s = torch.matmul(q[:, l].double().cuda().reshape(B, Hkv, -1, 128), K[:, :, :n].transpose(2, 3).contiguous()) / math.sqrt(128)
        near = s - s.amax(-1, keepdim=True)
        got = out[:, l, ..., :n] / out[:, l, ..., :n].gather(-1, s.argmax(-1, keepdim=True))
        off.append((got / near.exp() - 1)[(near > -0.5 * math.log(2)) & (near < 0)])
    off = torch.cat(off)
    assert len(off) > 2000 and float(off.square().mean().sqrt()) <= 3 * e


@pytest.mark.parametrize("L,H,Hkv,maxlen", [(1, 16, 4, 500), (1, 16, 4, 3000), (5, 4, 4, 700), (20, 4, 4, 300), (24, 4, 4, 4000), (40, 8, 4, 700), (70, 4, 2, 3000)])
def test_rows_behind_a_sequence_may_hold_anything(L, H, Hkv, maxlen):
    """the same bits whatever the rest of the capacity, and the rows that the call writes, held before: NaN, infinities, any bytes.  In one launch and three"""
    g = torch.Generator().manual_seed(L + maxlen)
    B, f = 5, _inv_freq().cuda()
    q, k, v = (x.cuda() for x in _random(g, B, L, H, Hkv))
    cache = _filled(g, 2, B, Hkv, maxlen)
    lengths, q_lens = torch.tensor([0, 31, 128, maxlen // 2 + 1, maxlen - L], dtype=torch.int32), torch.tensor([L, 1, L, max(L - 3, 0), L], dtype=torch.int32)
    held = torch.arange(maxlen) < lengths[:, None]
    written = (torch.arange(maxlen) < (lengths + q_lens)[:, None])[None, :, None, :, None].expand(2, -1, Hkv, -1, 80)
    fill = [torch.zeros_like(cache), torch.randint(-128, 128, cache.shape, generator=g, dtype=torch.int8)]
    for bad in (math.nan, math.inf, -math.inf, 65504.0):
        fill.append(torch.randint(-128, 128, cache.shape, generator=g, dtype=torch.int8))
        fill[-1][..., 64:] = torch.full((8,), bad, dtype=torch.float16).view(torch.int8)
    got = []
    for other in fill:
        dev = torch.where(held[None, :, None, :, None], cache, other).cuda()
        out = llmops.attention_rope_q4(q, k, v, f, dev, lengths.cuda(), 0, q_lens=q_lens.cuda())
        got.append((out, dev.cpu()))
        assert out.isfinite().all() and torch.equal(got[-1][1][~written], other[~written])  # (what is behind stays as it is)
    for out, dev in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(dev[written], got[0][1][written])
