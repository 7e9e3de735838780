"""verify_drafts against its definition, evaluated draft by draft in 64 bits on the host.  Answers are whole numbers and have to be
equal: inputs are such that no random number lies within 1e-12 of a border (checked on the host)."""
import math

import numpy as np
import pytest
import torch

import llmops

pytestmark = pytest.mark.gpu


def _weights(z, t):
    """w of a row; None if no logit is above minus infinity"""
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    top = z.max()
    if top == -np.inf:
        return None
    if top == np.inf:
        return (z == top).astype(np.float64)
    return np.exp((z - top) / np.float64(t))


def _reference(logits, drafts, uniforms, probs, temperature, lens):
    B, rows, V = logits.shape
    K = rows - 1
    tokens, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int32)
    for b in range(B):
        n = K if lens is None else min(max(int(lens[b]), 0), K)
        t = float(temperature[b])
        i, r, nothing = 0, None, False
        while True:
            z = logits[b, i]
            if not t > 0:
                z = np.where(np.isnan(z), -np.inf, z)
                best = int(z.argmax()) if z.max() > -np.inf else -1
                if i < n and drafts[b, i] == best and best >= 0:
                    tokens[b, i] = best
                    i += 1
                    continue
                nxt = best
                break
            w = _weights(z, t)
            if w is None:
                nxt = -1
                break
            p = w / w.sum()
            if i == n:
                r = p
            else:
                x = int(drafts[b, i])
                q = probs[b, i].astype(np.float64) if probs is not None else None
                if 0 <= x < V:
                    border = p[x] / (q[x] if q is not None else 1.0) if (q is None or q[x] > 0) else np.inf
                    # (a border of exactly 1, all the weight on one token, is exact on both sides)
                    assert border == 1.0 or not abs(float(uniforms[b, i]) - border) < 1e-12
                    if float(uniforms[b, i]) * (q[x] if q is not None else 1.0) < p[x]:
                        tokens[b, i] = x
                        i += 1
                        continue
                if q is not None:
                    d = p - q
                    r = np.where(d > 0, d, 0.0)
                else:
                    r = p.copy()
                    if 0 <= x < V:
                        r[x] = 0.0
                if not r.sum() > 0:
                    r = p
            c = np.cumsum(r)
            goal = float(uniforms[b, K]) * c[-1]
            above = np.nonzero(c > goal)[0]
            nxt = int(above[0]) if len(above) else int(np.nonzero(r)[0][-1])
            assert np.abs(c / c[-1] - float(uniforms[b, K])).min() > 1e-12 or float(uniforms[b, K]) in (0.0, 1.0)
            break
        tokens[b, i] = nxt
        accepted[b] = i
    return tokens, accepted


def _case(B, K, V, probs, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * spread
    q = torch.softmax(logits[:, :K] + 0.7 * torch.randn(B, K, V, generator=g), dim=-1) if probs else None
    if not K:
        drafts = torch.zeros(B, 0, dtype=torch.int64)
    elif probs:
        drafts = torch.multinomial(q.reshape(B * K, V), 1, generator=g).reshape(B, K)
    else:
        drafts = torch.where(torch.rand(B, K, generator=g) < 0.8, logits[:, :K].argmax(-1), torch.randint(0, V, (B, K), generator=g))
        logits[:, :K].scatter_add_(2, logits[:, :K].argmax(-1, keepdim=True), torch.full((B, K, 1), 6.0))
    return logits, drafts, torch.rand(B, K + 1, generator=g), q


def _check(logits, drafts, uniforms, q, temperature=None, lens=None):
    B = logits.shape[0]
    d = lambda x: x.cuda() if isinstance(x, torch.Tensor) else x  # noqa: E731
    tokens, accepted = llmops.verify_drafts(d(logits), d(drafts), d(uniforms), draft_probs=d(q), temperature=d(temperature), draft_lens=d(lens))
    t = temperature.numpy() if isinstance(temperature, torch.Tensor) else np.full(B, 1.0 if temperature is None else temperature, np.float32)
    want, n = _reference(logits.numpy(), drafts.numpy(), uniforms.numpy(), None if q is None else q.numpy(), t, lens)
    assert accepted.dtype == torch.int32 and tokens.dtype == torch.int64
    assert np.array_equal(accepted.cpu().numpy(), n), (accepted.cpu().numpy(), n)
    assert np.array_equal(tokens.cpu().numpy(), want), (tokens.cpu().numpy(), want)
    return n


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 1, 2), (1, 0, 1), (3, 0, 1000), (1, 4, 55296), (40, 3, 4096), (9, 7, 4097), (5, 2, 12289), (2, 300, 33), (130, 1, 50), (6, 5, 32003)])
def test_against_the_definition(B, K, V, probs):
    logits, drafts, uniforms, q = _case(B, K, V, probs and K > 0, seed=B + K)
    _check(logits, drafts, uniforms, q)
    t = torch.tensor([1.0, 0.7, 0.0, 1.3, -1.0, 0.02, math.nan])[torch.arange(B) % 7].contiguous()
    lens = torch.arange(B, dtype=torch.int32) % (K + 3) - 1  # (from -1 to K + 1: held to 0 .. K)
    _check(logits, drafts, uniforms, q, t, lens)
    _check(logits, drafts.to(torch.int32), uniforms, q, 0.8)
    _check(logits, drafts, uniforms, q, 0)


def test_some_are_accepted_and_some_not():
    logits, drafts, uniforms, q = _case(64, 4, 3000, True, seed=1)
    n = _check(logits, drafts, uniforms, q)
    assert set(n.tolist()) == {0, 1, 2, 3, 4}


def test_every_border_of_a_small_vocabulary():
    """random numbers over a grid: each token has its share, and a token without weight never comes"""
    V, G = 7, 4001
    z = torch.tensor([0.3, -math.inf, 1.0, math.nan, -2.0, 0.3, -math.inf])
    q = torch.tensor([0.5, 0.0, 0.1, 0.0, 0.1, 0.3, 0.0])
    u = (torch.arange(G) + 0.5) / G
    w = _weights(z.numpy(), 1.0)
    # drawn from the row itself
    tokens, _ = llmops.verify_drafts(z.expand(G, 1, V).contiguous().cuda(), torch.zeros(G, 0, dtype=torch.int64).cuda(), u[:, None].contiguous().cuda())
    share = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V) / G
    assert np.abs(share - w / w.sum()).max() <= 1.0 / G and share[[1, 3, 6]].sum() == 0
    # behind a refused draft (token 0, q > p)
    p = w / w.sum()
    r = np.maximum(p - q.numpy().astype(np.float64), 0)
    both = torch.stack((torch.full((G,), 0.999), u), dim=1)
    tokens, n = llmops.verify_drafts(z.expand(G, 2, V).contiguous().cuda(), torch.zeros(G, 1, dtype=torch.int64).cuda(), both.cuda(),
                                     draft_probs=q.expand(G, 1, V).contiguous().cuda())
    assert (n == 0).all() and (tokens[:, 1] == -1).all()
    share = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V) / G
    assert np.abs(share - r / r.sum()).max() <= 1.0 / G


def test_distribution_of_answers_is_the_models():
    """200 000 draws with drafts from another distribution: the first token's frequencies are p, not q"""
    n, V = 200000, 12
    g = torch.Generator().manual_seed(3)
    z = torch.randn(V, generator=g)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    drafts = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 2, generator=g)
    tokens, _ = llmops.verify_drafts(z.expand(n, 2, V).contiguous().cuda(), drafts.cuda(), u.cuda(), draft_probs=q.expand(n, 1, V).contiguous().cuda())
    share = np.bincount(tokens[:, 0].cpu().numpy(), minlength=V) / n
    p = torch.softmax(z.double(), 0).numpy()
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()  # (five standard deviations)


def test_rows_that_hold_little():
    V = 5000
    logits, drafts, uniforms, q = _case(12, 2, V, True, seed=7)
    logits[0] = -math.inf  # nothing
    logits[1, 0] = math.nan
    logits[2, 0, 17] = math.inf  # all of it, and not the draft
    logits[3, 0, 4500], logits[3, 0, 30] = math.inf, math.inf  # half each
    logits[4, 0, :4100] = -math.inf  # the first run empty
    logits[5, 0] = torch.finfo(torch.float32).min
    logits[6, 0, :] = 2.0  # all alike
    logits[7, 1] = -math.inf
    logits[7, 1, 4999] = -3.0
    drafts[8, 0], drafts[9, 0], drafts[10, 1] = -1, V, 1 << 40
    q[11, 0] = math.nan
    for t in (None, 0, 0.5):
        _check(logits, drafts, uniforms, q, t)
        _check(logits, drafts, uniforms, None, t)


def test_nothing_left_of_the_target():
    """q covers p entirely where a draft was refused: the next token comes from p"""
    logits, drafts, uniforms, _ = _case(6, 1, 900, True, seed=9)
    q = torch.ones(6, 1, 900)
    uniforms[:, 0] = 0.999999
    assert (_check(logits, drafts, uniforms, q) == 0).all()
    # the draft is all that there is, and the random number is out of its range
    logits = torch.full((2, 2, 10), -math.inf)
    logits[:, :, 4] = 1.0
    _check(logits, torch.full((2, 1), 4), torch.ones(2, 2), None)


def test_random_numbers_at_their_ends():
    logits, drafts, uniforms, q = _case(8, 3, 4200, True, seed=4)
    for u in (0.0, 1.0, float(np.nextafter(np.float32(1), np.float32(0)))):
        uniforms[:, 3] = u
        _check(logits, drafts, uniforms, q)


def test_lowest_of_equals():
    logits = torch.zeros(3, 2, 9000)
    logits[0, 0, [8000, 20, 5000]] = 1.0
    logits[1, 0, [4096, 4095]] = 2.0
    tokens, n = llmops.verify_drafts(logits.cuda(), torch.tensor([[20], [4096], [1]]).cuda(), torch.rand(3, 2).cuda(), temperature=0.0)
    assert n.tolist() == [1, 0, 0] and tokens.tolist() == [[20, 0], [4095, -1], [0, -1]]


def test_graph_and_streams():
    logits, drafts, uniforms, q = (t.cuda() for t in _case(6, 3, 6000, True, seed=5))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        llmops.verify_drafts(logits, drafts, uniforms, draft_probs=q)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = llmops.verify_drafts(logits, drafts, uniforms, draft_probs=q)
    torch.cuda.synchronize()
    for _ in range(5):
        uniforms.copy_((uniforms * 7.31) % 1.0)
        want = llmops.verify_drafts(logits, drafts, uniforms, draft_probs=q)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    logits, drafts, uniforms, q = (t.cuda() for t in _case(2, 3, 50, True, seed=1))
    n = torch.zeros(2, dtype=torch.int32).cuda()
    t = torch.ones(2).cuda()
    llmops.verify_drafts(logits, drafts, uniforms, draft_probs=q, temperature=t, draft_lens=n)
    for args, kw in (((logits.cpu(), drafts, uniforms), {}), ((logits.half(), drafts, uniforms), {}), ((logits[0], drafts, uniforms), {}),
                     ((logits, drafts.float(), uniforms), {}), ((logits, drafts[:, :2].contiguous(), uniforms), {}), ((logits, drafts, uniforms[:, :3].contiguous()), {}),
                     ((logits[..., ::2], drafts, uniforms), {}), ((logits, drafts, uniforms), dict(draft_probs=q[:, :2].contiguous())),
                     ((logits, drafts, uniforms), dict(draft_probs=q.double())), ((logits, drafts, uniforms), dict(temperature=t.double())),
                     ((logits, drafts, uniforms), dict(temperature=t[:1])), ((logits, drafts, uniforms), dict(draft_lens=n.long())),
                     ((logits, drafts, uniforms), dict(draft_lens=n[:1])), ((logits, drafts.cpu(), uniforms), {}), ((logits, drafts[:, ::2], uniforms), {})):
        with pytest.raises(RuntimeError):
            llmops.verify_drafts(*args, **kw)


def test_numbers_that_are_none_of_the_definitions():
    """random numbers and temperatures outside their ranges: still a token that weighs something"""
    logits, drafts, uniforms, q = _case(8, 3, 4200, True, seed=6)
    logits[:, :, :50] = -math.inf
    for bad in (math.nan, math.inf, -math.inf, -1.0, 2.0):
        for t in (None, math.inf, 1e-40, math.nan):
            for probs in (q.cuda(), None):
                u = uniforms.clone()
                u[::2], u[1, 3], u[3, 0] = bad, bad, bad
                tokens, n = llmops.verify_drafts(logits.cuda(), drafts.cuda(), u.cuda(), draft_probs=probs, temperature=t)
                tokens, n = tokens.cpu(), n.cpu()
                assert ((n >= 0) & (n <= 3)).all()
                last = tokens.gather(1, n[:, None].long())[:, 0]
                assert ((last >= 50) & (last < 4200)).all() and (tokens[torch.arange(4)[None] > n[:, None]] == -1).all()


def test_offsets_past_32_bits():
    """the last of many sequences whose logits are more than 2^31 values, beside the same sequence alone"""
    B, K, V = 64, 3, (1 << 23) + 5
    g = torch.Generator(device="cuda").manual_seed(12)
    logits, q = torch.zeros(B, K + 1, V, device="cuda"), torch.zeros(B, K, V, device="cuda")
    logits[B - 1] = torch.randn(K + 1, V, generator=g, device="cuda")
    q[B - 1] = torch.softmax(logits[B - 1, :K] + torch.randn(K, V, generator=g, device="cuda"), -1)
    drafts, uniforms = torch.randint(0, V, (B, K), generator=g, device="cuda"), torch.rand(B, K + 1, generator=g, device="cuda")
    for probs in (q, None):
        tokens, n = llmops.verify_drafts(logits, drafts, uniforms, draft_probs=probs)
        one, m = llmops.verify_drafts(logits[B - 1:], drafts[B - 1:], uniforms[B - 1:], draft_probs=None if probs is None else probs[B - 1:])
        assert torch.equal(tokens[B - 1:], one) and torch.equal(n[B - 1:], m)
