"""attention_rope_prefix against the formula in 64 bits: lengths, heads, cache types, padding, masked rows that hold anything, values
outside the halves' range, graphs and streams.

Tolerances.  A score is a sum of 128 products of a 22-bit and a 21-bit value, each product off by at most 2^-21 + 2^-22 of itself
(rounding errors of both factors) and summed in fp32; with values ~N(0, 1) a score is then off by about sqrt(128) * 2^-21 * 1/sqrt(128) +
fp32's own 128 roundings of partial sums ~ 10 (2^-24 * 10 * sqrt(128) / sqrt(128)), together about 1e-6, and a result, whose weights are
off by that, by about 1e-6 of itself: 4e-6 in the 2-norm, and 40 times a value's share for the largest of some 10^5 values."""
import math

import numpy as np
import pytest
import torch

import llmops

pytestmark = pytest.mark.gpu

S = 128
REL, MAX = 4e-6, 4e-5


def _inv_freq(half=64):
    return 1.0 / (10000.0 ** (torch.arange(0, half, dtype=torch.float32) / half))


def _reference(q, k, v, inv_freq, prefix, P, cache, lengths, q_lens, layer=0):
    """(out, cache) in 64 bits on the host; rows of `cache` (float64 copy) are filled with the new rows as they are"""
    B, L, width = q.shape
    Hkv, maxlen = cache.shape[2], cache.shape[3]
    H, half = width // S, inv_freq.shape[0]
    out = torch.zeros(B, L, H, S, dtype=torch.float64)
    f = inv_freq.double()

    def rot(x, pos):  # [L, heads, S]
        c, s = torch.cos(pos[:, None] * f)[:, None], torch.sin(pos[:, None] * f)[:, None]
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat((c * a - s * b, s * a + c * b, x[..., 2 * half:]), dim=-1)

    new = {}
    for b in range(B):
        n0 = min(max(int(lengths[b]), 0), maxlen)
        n = min(max(L if q_lens is None else min(int(q_lens[b]), L), 0), maxlen - n0)
        if n == 0:
            continue
        pos = torch.arange(P + n0, P + n0 + n, dtype=torch.float64)
        qq, kk = rot(q[b, :n].double().reshape(n, H, S), pos), rot(k[b, :n].double().reshape(n, Hkv, S), pos)
        new[b] = (n0, n, kk, v[b, :n].double().reshape(n, Hkv, S))
        own = cache[2 * layer:2 * layer + 2, b].double().clone()
        for h in range(H):
            hk = h // (H // Hkv)
            keys = torch.cat((prefix[2 * layer, 0, hk, :P].double(), own[0, hk, :n0 + n]))
            vals = torch.cat((prefix[2 * layer + 1, 0, hk, :P].double(), own[1, hk, :n0 + n]))
            for l in range(n):
                r = P + n0 + l + 1
                out[b, l, h] = torch.softmax(keys[:r] @ qq[l, h] / math.sqrt(S), 0) @ vals[:r]
    return out.reshape(B, L, width), new


def _case(B, L, H, Hkv, P, maxlen, half_cache, seed, lengths=None, q_lens=None, layers=1, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    t = torch.float16 if half_cache else torch.float32
    qkv = torch.randn(B, L, (H + 2 * Hkv) * S, generator=g)
    prefix = (torch.randn(2 * layers, 1, Hkv, max(P, 1) + 3, S, generator=g) * scale).to(t)
    cache = (torch.randn(2 * layers, B, Hkv, maxlen, S, generator=g) * scale).to(t)
    if lengths is None:
        lengths = torch.randint(0, maxlen - L + 1, (B,), generator=g)
    return qkv, prefix, cache, torch.as_tensor(lengths, dtype=torch.int32), None if q_lens is None else torch.as_tensor(q_lens, dtype=torch.int32)


def _split(qkv, H, Hkv):
    return qkv[..., :H * S], qkv[..., H * S:(H + Hkv) * S], qkv[..., (H + Hkv) * S:]


def _call(qkv, H, Hkv, f, prefix, P, cache, lengths, q_lens, layer=0):
    d = lambda x: None if x is None else x.cuda()  # noqa: E731
    kv = cache.cuda()
    out = llmops.attention_rope_prefix(*_split(d(qkv), H, Hkv), d(f), d(prefix), P, kv, d(lengths), layer, q_lens=d(q_lens))
    return out, kv


def _check(qkv, H, Hkv, prefix, P, cache, lengths, q_lens, layer=0, f=None, rel=REL, top=MAX):
    f = _inv_freq() if f is None else f
    out, kv = _call(qkv, H, Hkv, f, prefix, P, cache, lengths, q_lens, layer)
    out, kv = out.cpu(), kv.cpu()
    ref, new = _reference(*_split(qkv, H, Hkv), f, prefix, P, kv, lengths, q_lens, layer)  # (on the rows as the cache holds them)
    # the cache: new rows rotated, everything else as it was
    want = cache.clone()
    for b, (n0, n, kk, vv) in new.items():
        for plane, rows in ((0, kk), (1, vv)):
            got = kv[2 * layer + plane, b, :, n0:n0 + n].double()
            rows = rows.transpose(0, 1)
            step = torch.finfo(cache.dtype).eps / 2 if cache.dtype == torch.float16 else 0.0
            # a rotation: two products and a sum in fp32, cos and sin off by 2^-22 at most
            assert ((got - rows).abs() <= rows.abs() * step + 6e-7 * rows.abs().max() + 3e-8).all()
            want[2 * layer + plane, b, :, n0:n0 + n] = kv[2 * layer + plane, b, :, n0:n0 + n]
    assert torch.equal(want.view(torch.int16 if cache.dtype == torch.float16 else torch.int32),
                       kv.view(torch.int16 if cache.dtype == torch.float16 else torch.int32))
    live = torch.zeros(out.shape[:2], dtype=torch.bool)
    for b, (n0, n, _, _) in new.items():
        live[b, :n] = True
    assert (out[~live] == 0).all()
    if live.any():
        err = (out.double() - ref)[live]
        assert err.norm() <= rel * ref.norm(), (err.norm() / ref.norm())
        assert err.abs().max() <= top * ref.abs().max()
    return out, kv


SIZES = [  # B, tokens, H, Hkv, prefix, own rows
    (1, 1, 2, 2, 0, 1), (1, 1, 4, 1, 5, 40), (3, 1, 4, 4, 127, 64), (2, 1, 8, 2, 129, 300), (5, 3, 4, 2, 260, 33),
    (2, 17, 4, 4, 64, 70), (1, 40, 4, 2, 31, 90), (3, 33, 2, 1, 100, 140), (17, 1, 2, 2, 512, 20), (40, 2, 2, 1, 300, 9),
    (2, 130, 2, 2, 70, 200), (1, 300, 4, 1, 0, 300), (2, 65, 6, 3, 33, 200), (1, 1, 1, 1, 2000, 1500), (70, 1, 2, 1, 33, 5), (4, 16, 8, 1, 96, 32),
]


@pytest.mark.parametrize("half_cache", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,P,maxlen", SIZES)
def test_against_64_bits(B, L, H, Hkv, P, maxlen, half_cache):
    case = _case(B, L, H, Hkv, P, maxlen, half_cache, seed=B * 1000 + L)
    _check(case[0], H, Hkv, case[1], P, case[2], case[3], None)


@pytest.mark.parametrize("half_cache", [False, True])
@pytest.mark.parametrize("L,H,Hkv,P", [(5, 4, 2, 50), (5, 4, 4, 0), (20, 8, 1, 200), (150, 2, 2, 40)])
def test_padding_and_lengths_that_do_not_fit(L, H, Hkv, P, half_cache):
    maxlen = L + 30
    lengths = [0, 3, maxlen - L, maxlen - L + 2, maxlen - 1, maxlen, maxlen + 7, -4, 30]
    q_lens = [L, 0, L - 1, L, L, L, 1, 2, L + 9]
    case = _case(len(lengths), L, H, Hkv, P, maxlen, half_cache, seed=5, lengths=lengths, q_lens=q_lens)
    _check(case[0], H, Hkv, case[1], P, case[2], case[3], case[4])


@pytest.mark.parametrize("half", [1, 7, 10, 32, 64])
def test_partial_rotation(half):
    case = _case(3, 4, 4, 2, 77, 40, False, seed=half)
    _check(case[0], 4, 2, case[1], 77, case[2], case[3], None, f=_inv_freq(half))


def test_second_layer_and_far_positions():
    case = _case(2, 3, 2, 1, 9001, 6000, True, seed=3, layers=2, lengths=[5990, 17])
    _check(case[0], 2, 1, case[1], 9001, case[2], case[3], None, layer=1)


@pytest.mark.parametrize("L,P", [(1, 40), (4, 40), (70, 40), (1, 700), (40, 0)])
@pytest.mark.parametrize("half_cache", [False, True])
def test_masked_rows_hold_anything(L, P, half_cache):
    """rows behind a sequence's own, rows of the prefix behind its length, other sequences and padding: no effect, bit for bit;
    a later token's NaN stays with the tokens that see it"""
    H, Hkv, B, maxlen = 4, 2, 3, 200
    qkv, prefix, cache, lengths, q_lens = _case(B, L, H, Hkv, P, maxlen, half_cache, seed=11, lengths=[0, 50, 128], q_lens=[L, max(1, L - 1), L])
    f = _inv_freq()
    want, kv = _call(qkv, H, Hkv, f, prefix, P, cache, lengths, q_lens)
    bad = cache.clone()
    for b in range(B):
        for at, x in enumerate((math.nan, math.inf, -math.inf, torch.finfo(cache.dtype).min)):
            bad[:, b, :, int(lengths[b]) + int(q_lens[b]) + at::4] = x
    dirty, pre = qkv.clone(), prefix.clone()
    dirty[1, int(q_lens[1]):] = math.nan
    pre[:, :, :, P:] = math.nan
    got, kv2 = _call(dirty, H, Hkv, f, pre, P, bad, lengths, q_lens)
    assert torch.equal(got, want)
    for b in range(B):
        n = int(lengths[b]) + int(q_lens[b])
        assert torch.equal(kv2[:, b, :, :n], kv[:, b, :, :n])
    if L > 1:  # v of the last token is NaN: the tokens before it are as they were
        dirty = qkv.clone()
        dirty[0, L - 1, (H + Hkv) * S:] = math.nan
        dirty[2, L - 1, H * S:] = math.inf
        got, _ = _call(dirty, H, Hkv, f, prefix, P, cache, lengths, q_lens)
        for b in (0, 2):
            assert torch.isfinite(got[b, :L - 1]).all() and not torch.isfinite(got[b, L - 1]).any()
            ref = want[b, :L - 1]
            assert (got[b, :L - 1] - ref).abs().max() <= MAX * ref.abs().max()
        assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("L,P", [(1, 300), (3, 90), (70, 90)])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1e-3, 1e-3, 1e3), (1e5, 1e6, 1e-5), (1.0, 1e12, 1.0), (3e4, 3e4, 1e-4), (1e-6, 1.0, 1e6)])
def test_magnitudes(L, P, kscale, vscale, qscale):
    qkv, prefix, cache, lengths, _ = _case(2, L, 4, 2, P, L + 60, False, seed=2)
    qkv[..., :4 * S] *= qscale
    for t in (prefix, cache):
        t[0] *= kscale
        t[1] *= vscale
    qkv[..., 4 * S:6 * S] *= kscale
    qkv[..., 6 * S:] *= vscale
    _check(qkv, 4, 2, prefix, P, cache, lengths, None)


def test_infinite_and_nan_queries_and_keys():
    qkv, prefix, cache, lengths, _ = _case(3, 2, 2, 2, 40, 30, False, seed=8, lengths=[3, 4, 5])
    want, _ = _call(qkv, 2, 2, _inv_freq(), prefix, 40, cache, lengths, None)
    qkv[1, 0, 5] = math.nan  # a query's head
    got, _ = _call(qkv, 2, 2, _inv_freq(), prefix, 40, cache, lengths, None)
    assert torch.isnan(got[1, 0, :S]).all()
    got[1, 0, :S] = want[1, 0, :S] = 0
    assert torch.equal(got, want)
    cache[0, 2, 1, 2, 7] = math.nan  # a key that sequence 2 sees with head 1
    got, _ = _call(qkv, 2, 2, _inv_freq(), prefix, 40, cache, lengths, None)
    assert torch.isnan(got[2, :, S:]).all()
    got[1, 0, :S] = 0
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[2, :, :S], want[2, :, :S])


def test_a_prefix_from_attention_rope2_and_the_same_answers():
    """a prompt of 48 tokens through attention_rope2, its cache as the prefix; then each sequence's turn, token by token and at once,
    against attention_rope2 on a cache that holds both"""
    H, P, L, maxlen, f = 4, 48, 6, 20, _inv_freq().cuda()
    g = torch.Generator().manual_seed(1)
    x = [torch.randn(1, P, H * S, generator=g).cuda() for _ in range(3)]
    prefix = torch.zeros(2, 1, H, 64, S).cuda()
    llmops.attention_rope2(*(t.clone() for t in x), f, prefix, torch.arange(P, dtype=torch.int32).cuda(), 0, 0)
    turns = [torch.randn(2, L, H * S, generator=g).cuda() for _ in range(3)]
    want = []
    for b in range(2):
        cache = torch.zeros(2, 1, H, P + L, S).cuda()
        cache[:, :, :, :P] = prefix[:, :, :, :P]
        q, k, v = (t[b:b + 1].clone() for t in turns)
        llmops.attention_rope2(q, k, v, f, cache, torch.arange(P, P + L, dtype=torch.int32).cuda(), P, 0)
        want.append(q)
    want = torch.cat(want)
    kv = torch.zeros(2, 2, H, maxlen, S).cuda()
    lengths = torch.zeros(2, dtype=torch.int32).cuda()
    at_once = llmops.attention_rope_prefix(*turns, f, prefix, P, kv, lengths, 0)
    kv.zero_()
    steps = []
    for l in range(L):
        steps.append(llmops.attention_rope_prefix(*(t[:, l:l + 1] for t in turns), f, prefix, P, kv, lengths, 0))
        lengths += 1
    # (attention_rope2's angles are products in fp32: at position 54 off by up to 54 * 2^-24 = 3e-6)
    for got in (at_once, torch.cat(steps, dim=1)):
        assert (got - want).abs().max() <= 2e-5 * want.abs().max()


def test_same_bits_and_layouts():
    qkv, prefix, cache, lengths, _ = _case(4, 3, 4, 2, 333, 90, False, seed=6)
    f = _inv_freq().cuda()
    q, k, v = _split(qkv.cuda(), 4, 2)
    first, kv = _call(qkv, 4, 2, f, prefix, 333, cache, lengths, None)
    for form in (lambda t: t, lambda t: t.contiguous(), lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        kv2 = cache.cuda()
        got = llmops.attention_rope_prefix(form(q), form(k), form(v), f, prefix.cuda(), 333, kv2, lengths.cuda(), 0)
        assert torch.equal(got, first) and torch.equal(kv2, kv)


@pytest.mark.parametrize("L", [1, 40])
def test_graph_serves_following_steps(L):
    qkv, prefix, cache, lengths, _ = _case(3, L, 4, 2, 100, 4 * L + 9, True, seed=9, lengths=[0, 1, 5])
    f, prefix = _inv_freq().cuda(), prefix.cuda()
    q, k, v = (t.contiguous() for t in _split(qkv.cuda(), 4, 2))
    n = lengths.cuda()
    kv, kv_eager = cache.cuda(), cache.cuda()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        llmops.attention_rope_prefix(q, k, v, f, prefix, 100, kv.clone(), n, 0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = llmops.attention_rope_prefix(q, k, v, f, prefix, 100, kv, n, 0)
    torch.cuda.synchronize()
    for step in range(4):
        q.copy_(q.roll(1, dims=2))
        want = llmops.attention_rope_prefix(q, k, v, f, prefix, 100, kv_eager, n, 0)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kv, kv_eager)
        n += L
        torch.cuda.synchronize()


def test_two_streams_at_once():
    cases = [_case(8, 2, 4, 2, 400, 300, False, seed=s) for s in (1, 2)]
    f = _inv_freq().cuda()
    args = [[t.contiguous() for t in _split(c[0].cuda(), 4, 2)] + [f, c[1].cuda(), 400] for c in cases]
    rest = [(c[2].cuda(), c[3].cuda()) for c in cases]
    want = [llmops.attention_rope_prefix(*a, *r, 0) for a, r in zip(args, rest)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(llmops.attention_rope_prefix(*args[i], *rest[i], 0))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals():
    qkv, prefix, cache, lengths, _ = _case(2, 2, 4, 2, 10, 8, False, seed=1)
    f, prefix, cache, n = _inv_freq().cuda(), prefix.cuda(), cache.cuda(), lengths.cuda()
    q, k, v = _split(qkv.cuda(), 4, 2)

    def call(**kw):
        a = dict(q=q, k=k, v=v, inv_freq=f, prefix_cache=prefix, prefix_len=10, kv_cache=cache, lengths=n, layer_id=0)
        a.update(kw)
        return llmops.attention_rope_prefix(**a)

    call()
    before = cache.clone()
    for kw in (dict(prefix_len=14), dict(prefix_len=-1), dict(layer_id=1), dict(layer_id=-1), dict(q=q.cpu()), dict(q=q.half()), dict(k=q), dict(q=q[..., 1:]),
               dict(q=q[..., 4:].contiguous()), dict(kv_cache=cache.half()), dict(kv_cache=cache.transpose(1, 2)), dict(prefix_cache=prefix.expand(2, 2, -1, -1, -1)),
               dict(lengths=n.long()), dict(lengths=n[:1]), dict(lengths=n.cpu()), dict(q_lens=n[:1]), dict(prefix_cache=None), dict(inv_freq=torch.ones(65).cuda()),
               dict(q=torch.zeros(2, 2, 4 * S + 1).cuda()[..., 1:]), dict(q=q[:1]), dict(kv_cache=cache[:, :, :, :, :64].contiguous())):
        with pytest.raises(RuntimeError):
            call(**kw)
    one = cache[:, :1].contiguous()
    with pytest.raises(RuntimeError, match="p1 <= o0"):  # the prefix inside the batch's own cache
        llmops.attention_rope_prefix(q[:1], k[:1], v[:1], f, one, 4, one, n[:1], 0)
    assert torch.equal(cache, before)


def test_offsets_past_32_bits():
    """the last of many sequences in a cache whose planes hold more than 2^31 values, beside the same sequence alone"""
    B, H, maxlen, n, P = 40, 8, 65536, 65534, 70
    g = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (torch.randn(B, 2, H * S, generator=g, device="cuda") for _ in range(3))
    prefix = torch.randn(2, 1, H, P, S, generator=g, device="cuda").half()
    alone = torch.randn(2, 1, H, maxlen, S, generator=g, device="cuda").half()
    kv = torch.empty(2, B, H, maxlen, S, dtype=torch.float16, device="cuda")
    kv[:, B - 1] = alone[:, 0]
    lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
    lengths[B - 1] = n
    f = _inv_freq().cuda()
    out = llmops.attention_rope_prefix(q, k, v, f, prefix, P, kv, lengths, 0)
    one = llmops.attention_rope_prefix(q[B - 1:], k[B - 1:], v[B - 1:], f, prefix, P, alone, lengths[B - 1:], 0)
    assert torch.equal(kv[:, B - 1], alone[:, 0])
    err = (out[B - 1] - one[0]).double()  # (each is off by REL at most)
    assert err.norm() <= 2 * REL * one.double().norm() and err.abs().max() <= 2 * MAX * one.abs().max()
    assert out.isfinite().all()


# one for each way that the work is cut up: all rows in one go; pieces, in one launch and in two; 32 queries to a workgroup; rows cut up for 64 and
# for 128 queries; a sequence's 64 and 128 queries in one sweep
KINDS = [(9, 2, 4, 2, 60, 40), (3, 2, 4, 2, 600, 40), (16, 1, 32, 32, 600, 9), (20, 1, 16, 16, 400, 9), (50, 2, 32, 8, 300, 9), (70, 1, 32, 32, 1100, 9),
         (3, 50, 2, 2, 100, 60), (64, 70, 8, 8, 70, 80)]


@pytest.mark.parametrize("half_cache", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,P,maxlen", KINDS)
def test_every_way_of_cutting_up(B, L, H, Hkv, P, maxlen, half_cache):
    qkv, prefix, cache, lengths, _ = _case(B, L, H, Hkv, P, maxlen, half_cache, seed=21)
    out, _ = _check(qkv, H, Hkv, prefix, P, cache, lengths, None)
    # what is behind the prefix and behind a sequence's rows has no effect, bit for bit
    pre, own = prefix.clone(), cache.clone()
    pre[:, :, :, P:] = math.nan
    for b in range(B):
        own[:, b, :, int(lengths[b]) + L:] = math.nan
    got, _ = _call(qkv, H, Hkv, _inv_freq(), pre, P, own, lengths, None)
    assert torch.equal(got.cpu(), out)
    # values that the halves do not hold, and then padding
    big = qkv.clone()
    big[..., H * S:] *= 1e5 if not half_cache else 1.0
    big[..., (H + Hkv) * S:] *= 1e2
    big[..., :H * S] *= 1e-5 if not half_cache else 1.0
    _check(big, H, Hkv, prefix, P, cache, lengths, (torch.arange(B) % (L + 1)).to(torch.int32))


@pytest.mark.parametrize("half_cache", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,P,maxlen", KINDS)
def test_queries_down_to_the_least_number(B, L, H, Hkv, P, maxlen, half_cache):
    """queries of 1e-36 down to the least denormal, tokens and heads of each beside each other and beside ordinary ones, in front of tiles that a
    mask ends in: their scores are 0 to 64 bits' eyes and an output is the mean of the rows seen"""
    qkv, prefix, cache, lengths, _ = _case(B, L, H, Hkv, P, maxlen, half_cache, seed=22)
    sizes = torch.tensor([1.0, 1e-36, 1e-38, 1e-39, 3e-41, 5e-42, 1e-43, 5e-45, 1.5e-45, 0.0])
    size = sizes[torch.arange(B * L * H) % len(sizes)].reshape(B, L, H, 1)
    qkv[..., :H * S] = (qkv[..., :H * S].reshape(B, L, H, S) * size).reshape(B, L, H * S)
    _check(qkv, H, Hkv, prefix, P, cache, lengths, None)


@pytest.mark.parametrize("L,P", [(1, 20), (1, 300), (3, 90), (70, 90)])
@pytest.mark.parametrize("q_size", [1e-37, 1e-39, 1e-41])
def test_least_queries_and_largest_keys(L, P, q_size):
    """A query's denormal is a multiple of 2^-149, and so are the rounding errors of its rotation and of its operands, 2^-148 at most: beside keys of
    3e37 = 2^124.5 a score is off by 2^-148 * 2^124.5 * sqrt(128) / sqrt(128) = 2^-23.5, within REL"""
    qkv, prefix, cache, lengths, _ = _case(2, L, 4, 2, P, L + 60, False, seed=23)
    qkv[..., :4 * S] *= q_size
    qkv[..., 4 * S:6 * S] *= 3e37
    prefix[0] *= 3e37
    cache[0] *= 3e37
    _check(qkv, 4, 2, prefix, P, cache, lengths, None)


# (tokens, prefix, rows of its own): odd positions, for which a product with a frequency is rounded in fp32
@pytest.mark.parametrize("L,P,n", [(1, 40001, 3), (1, 131071, 3), (20, 131071, 70), (70, 262139, 33), (2, 1000003, 5), (20, 70, 1000003), (3, 0, (1 << 24) - 3),
                                   (17, (1 << 24) - 60, 40), (60, (1 << 24) - 70, 9)])
def test_far_positions(L, P, n):
    """Keys (1, 0) in every pair of dimensions leave the cosines and sines of their positions in the cache.  Each is off by sincosf's 2 ulp (2^-23) and
    by the rounding of what is put back and of the product (2^-24 each): 2.4e-7.
    Rows before them are all alike, so that the sums have a closed form.  A score, at most ln(2^24) = 17, is off by 2 * 2.4e-7 of itself (both sides'
    rotation), 2^-21 + 2^-22 (operands) and 10 * 2^-24 (sums), 1.8e-6, that is 3e-5; a weight by a quarter of that, beside outputs near 1: 2e-5"""
    H, maxlen, f = 2, n + L, _inv_freq()
    N = P + n
    g = torch.Generator().manual_seed(L)
    a = math.log(N) * math.sqrt(S) / 64  # (a token's own row weighs as much as all before it)
    pair = torch.cat((torch.ones(64), torch.zeros(64)))
    q, k, v = (a * pair).repeat(H).expand(1, L, -1).contiguous(), pair.expand(1, L, -1).contiguous(), torch.randn(1, L, S, generator=g)
    key, value = 2.0 ** -9, 0.25
    prefix = torch.empty(2, 1, 1, P, S, device="cuda") if P else None
    kv = torch.empty(2, 1, 1, maxlen, S, device="cuda")
    for t in (prefix, kv):
        if t is not None:
            t[0], t[1] = key, value
    out = llmops.attention_rope_prefix(q.cuda(), k.cuda(), v.cuda(), f.cuda(), prefix, P, kv, torch.tensor([n], dtype=torch.int32).cuda(), 0)
    angle = torch.arange(N, N + L, dtype=torch.float64)[:, None] * f.double()
    turned = torch.cat((angle.cos(), angle.sin()), dim=1)
    rows = kv[0, 0, 0, n:].cpu().double()
    assert (rows - turned).abs().max() <= 2.4e-7, (rows - turned).abs().max()
    assert torch.equal(kv[1, 0, 0, n:].cpu(), v[0])
    scores = (a * turned) @ turned.T / math.sqrt(S)
    before = (a * turned).sum(1, keepdim=True) * key / math.sqrt(S)
    weights = torch.cat((before + math.log(N), scores.masked_fill(torch.ones(L, L).triu(1) > 0, -math.inf)), dim=1).softmax(1)
    want = weights[:, :1] * value + weights[:, 1:] @ v[0].double()
    for h in range(H):
        err = out[0, :, h * S:(h + 1) * S].cpu().double() - want
        assert err.norm() <= 2e-5 * want.norm() and err.abs().max() <= 2e-4 * want.abs().max(), (err.norm() / want.norm(), err.abs().max())


@pytest.mark.parametrize("L,P", [(1, 20), (1, 300), (3, 90), (40, 90), (70, 90)])
@pytest.mark.parametrize("kscale,vscale,qscale", [(1.0, 1e-6, 1.0), (1.0, 1e-7, 1.0), (1e-6, 1.0, 1e6), (1e-7, 1e-7, 1e7)])
def test_halves_below_their_normal_range(L, P, kscale, vscale, qscale):
    """caches of halves that hold denormals only: within REL of the largest output like all others"""
    qkv, prefix, cache, lengths, _ = _case(2, L, 4, 2, P, L + 60, True, seed=24)
    qkv[..., :4 * S] *= qscale
    for t in (prefix, cache):
        t[0], t[1] = (t[0].float() * kscale).half(), (t[1].float() * vscale).half()
    qkv[..., 4 * S:6 * S] *= kscale
    qkv[..., 6 * S:] *= vscale
    _check(qkv, 4, 2, prefix, P, cache, lengths, None)


def test_inputs_over_the_new_rows_are_refused():
    qkv, prefix, cache, lengths, _ = _case(2, 2, 4, 2, 10, 8, False, seed=1, layers=2)
    q, k, v = (t.contiguous() for t in _split(qkv.cuda(), 4, 2))
    f, prefix, cache, n = _inv_freq().cuda(), prefix.cuda(), cache.cuda(), lengths.cuda()
    before = cache.clone()
    inside = cache[0].flatten()[:2 * 2 * 2 * S].view(2, 2, 2 * S)
    for kw in (dict(k=inside), dict(v=inside), dict(q=cache[1].flatten()[:2 * 2 * 4 * S].view(2, 2, 4 * S))):
        with pytest.raises(RuntimeError, match="apart"):
            llmops.attention_rope_prefix(**{**dict(q=q, k=k, v=v, inv_freq=f, prefix_cache=prefix, prefix_len=10, kv_cache=cache, lengths=n, layer_id=0), **kw})
    assert torch.equal(cache, before)
    # the other layer's planes are nobody's now
    k2 = cache[2].flatten()[:2 * 2 * 2 * S].view(2, 2, 2 * S)
    want = llmops.attention_rope_prefix(q, k2.clone(), v, f, prefix, 10, cache.clone(), n, 0)
    assert torch.equal(llmops.attention_rope_prefix(q, k2, v, f, prefix, 10, cache, n, 0), want)
