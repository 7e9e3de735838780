"""token_logprobs against its definition in 64 bits on the host.

What fp32 may be off by, with e = 2^-24, t = z - max and w = exp(t): a weight by (2 |t| + 2) e of itself (the product with log2 e, exp2), sums of up to 32
weights to a thread, then over 64 lanes and 4 waves, by 40 e; so log S by (2 mean|t| + 42) e.  The sum of w t likewise, each product by e more.  Joining and logarithms are in 64 bits; results
are rounded once."""
import math

import numpy as np
import pytest
import torch

import llmops

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def _reference(z, tokens, top):
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    R, V = z.shape
    logprob, entropy, tol, etol = np.zeros(R), np.zeros(R), np.zeros(R), np.zeros(R)
    ids, lps = np.zeros((R, top), np.int64), np.zeros((R, top))
    for r in range(R):
        M = z[r].max()
        if M == -np.inf:
            lp = np.full(V, np.nan)
            t = w = np.zeros(V)
        elif M == np.inf:
            lp = np.where(z[r] == np.inf, -np.log((z[r] == np.inf).sum()), -np.inf)
            t, w = np.zeros(V), (z[r] == np.inf).astype(float)
        else:
            t = z[r] - M
            w = np.exp(t)
            lp = t - np.log(w.sum())
            t = np.where(w > 0, t, 0.0)
        p = w / max(w.sum(), 1e-300)
        entropy[r] = -(p[p > 0] * lp[p > 0]).sum() if M > -np.inf else np.nan
        logprob[r] = lp[tokens[r]] if 0 <= tokens[r] < V else 0.0
        mean = (p * -t).sum()
        tol[r] = (2 * mean + 42) * E
        etol[r] = tol[r] + (p * -t * (2 * -t + 43)).sum() * E + mean * tol[r]
        order = np.argsort(-z[r], kind="stable")[:top]
        ids[r], lps[r] = order, lp[order]
    return logprob, entropy, ids, lps, tol, etol


def _near(got, want, tol):
    got = got.cpu().double().numpy()
    plain = np.isfinite(want)
    assert np.array_equal(got[~plain], want[~plain], equal_nan=True)
    off = np.abs(got[plain] - want[plain])
    room = (np.broadcast_to(tol, want.shape) + np.abs(np.where(plain, want, 0.0)) * E + 1e-45)[plain]
    assert (off <= room).all(), (off.max(), (off / room).max())


def _check(logits, tokens, top):
    B, L, V = logits.shape
    lp, ent, ids, lps = llmops.token_logprobs(logits.cuda() if not logits.is_cuda else logits, tokens.cuda() if not tokens.is_cuda else tokens, top)
    assert lp.shape == ent.shape == (B, L) and ids.shape == lps.shape == (B, L, top) and ids.dtype == torch.int64
    w = _reference(logits.cpu().reshape(B * L, V).numpy(), tokens.cpu().reshape(-1).numpy(), top)
    _near(lp.flatten(), w[0], w[4])
    _near(ent.flatten(), w[1], w[5])
    assert np.array_equal(ids.cpu().numpy().reshape(B * L, top), w[2])
    _near(lps.reshape(B * L, top), w[3], w[4][:, None])


def _case(B, L, V, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, L, V, generator=g) * spread, torch.randint(0, V, (B, L), generator=g)


@pytest.mark.parametrize("top", [0, 1, 5, 20, 64])
@pytest.mark.parametrize("B,L,V", [(1, 1, 1), (1, 1, 64), (2, 3, 100), (1, 1, 55296), (3, 5, 2048), (3, 5, 2049), (2, 2, 32003), (40, 5, 8192), (150, 1, 8193), (1030, 1, 777), (5, 60, 9001)])
def test_against_the_definition(B, L, V, top):
    logits, tokens = _case(B, L, V, seed=V + top)
    tokens[0, 0] = -1 if top == 5 else tokens[0, 0]  # padding
    tokens[-1, -1] = V if top == 20 else tokens[-1, -1]
    _check(logits, tokens, min(top, V))


@pytest.mark.parametrize("V", [50, 2048, 5000, 20000])
def test_equal_logits_in_their_order(V):
    g = torch.Generator().manual_seed(V)
    rows = torch.zeros(8, 1, V)
    rows[1] = torch.randint(0, 3, (V,), generator=g).float()
    rows[2] = torch.arange(V).float() * 1e-3
    rows[3] = -torch.arange(V).float() * 1e-3
    rows[4] = (torch.arange(V) % 256 == 7).float() * 9
    rows[5, 0, ::1024] = 5.0
    rows[6] = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)  # (zeros of both signs are equal)
    rows[7, 0, V // 2:] = 1.0
    tokens = torch.randint(0, V, (8, 1), generator=g)
    for top in (1, 20, 50):
        _check(rows, tokens, top)


def test_infinities_and_nan():
    inf, nan = math.inf, math.nan
    for V in (70, 3000, 9000):
        g = torch.Generator().manual_seed(V)
        rows = torch.randn(9, 1, V, generator=g)
        rows[0] = -inf
        rows[1] = nan
        rows[2, 0, 5] = inf
        rows[3, 0, [3, V - 1, V // 2]] = inf
        rows[4, 0, ::2] = -inf
        rows[5, 0, ::3] = nan
        rows[6, 0, 1:] = -inf
        rows[7] = -inf
        rows[7, 0, V - 1] = 3.0
        rows[8] = torch.randn(V, generator=g) * 1e30
        tokens = torch.tensor([0, 1, 5, V - 1, 4, 3, 0, V - 1, int(rows[8].argmax())])[:, None]
        _check(rows, tokens, 7)
        _check(rows, torch.full_like(tokens, 6), 64)


@pytest.mark.parametrize("V", [70, 2048, 8195, 24000])
def test_few_tokens_are_allowed(V):
    g = torch.Generator().manual_seed(V)
    few = [n for n in (1, 5, 19, 20, 21, 63, 64, 65, 130, 300, 3000) if n <= V]
    rows = torch.full((4 * len(few), 1, V), -math.inf)
    for i, n in enumerate(few):
        x = torch.randn(n, generator=g)
        rows[4 * i, 0, torch.randperm(V, generator=g)[:n]] = x
        rows[4 * i + 1, 0, :n] = x
        rows[4 * i + 2, 0, V - n:] = x
        rows[4 * i + 3, 0, (torch.arange(n) * 4 % V)] = 1.0  # (equal ones)
    tokens = torch.randint(0, V, (len(rows), 1), generator=g)
    for top in (1, 20, 64):
        _check(rows, tokens, top)


@pytest.mark.parametrize("spread", [1e-3, 30.0, 1000.0])
def test_flat_and_steep(spread):
    logits, tokens = _case(6, 2, 4000, 5, spread)
    _check(logits, tokens, 10)
    _check(logits + 1e4, logits.argmax(-1), 10)


def test_a_text_against_the_logits_before_each_token():
    logits, ids = _case(3, 40, 1001, 6)
    logits, ids = logits.cuda(), ids.cuda()
    _check(logits[:, :-1], ids[:, 1:], 4)
    wide = torch.randn(3, 40, 2050, generator=torch.Generator().manual_seed(7)).cuda()
    _check(wide[..., 3:1004], ids.to(torch.int32), 4)
    _check(wide[:, ::3, 7:1010].transpose(0, 1), ids[:, ::3].T, 0)


def test_a_text_of_one_token_has_none_behind_it():
    logits, tokens = (x.cuda() for x in _case(3, 1, 50, 2))
    lp, ent, ids, lps = llmops.token_logprobs(logits[:, :-1], tokens[:, 1:], 4)
    assert lp.shape == ent.shape == (3, 0) and ids.shape == lps.shape == (3, 0, 4)
    with pytest.raises(RuntimeError):
        llmops.token_logprobs(logits[:, :-1], tokens[:, 1:], 51)


def test_offsets_past_32_bits():
    V = 1 << 20
    logits = torch.zeros(2100, V, device="cuda")  # 8.8 GB
    logits[2050, 777] = 5.0
    lp, ent, ids, lps = llmops.token_logprobs(logits[None, 2048:], torch.full((1, 52), 777, device="cuda"), 2)
    want = 5.0 - math.log(V - 1 + math.exp(5.0))
    assert abs(float(lp[0, 2]) - want) < 42 * E + 14 * E and ids[0, 2].tolist() == [777, 0] and ids[0, 3].tolist() == [0, 1]


def test_captured():
    logits, tokens = (x.cuda() for x in _case(4, 3, 20000, 8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        llmops.token_logprobs(logits, tokens, 9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = llmops.token_logprobs(logits, tokens, 9)
    g = torch.Generator().manual_seed(9)
    for _ in range(4):
        torch.cuda.synchronize()
        logits.copy_(torch.randn(logits.shape, generator=g) * 2), tokens.copy_(torch.randint(0, 20000, tokens.shape, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, llmops.token_logprobs(logits, tokens, 9)))


def test_refusals():
    logits, tokens = (x.cuda() for x in _case(2, 3, 100, 1))
    for a in ((logits.half(), tokens, 0), (logits, tokens[:1], 0), (logits, tokens.float(), 0), (logits, tokens, 65), (logits, tokens, -1), (logits[..., :30], tokens, 31),
              (logits[..., ::2], tokens, 0), (logits.cpu(), tokens, 0), (logits, tokens.cpu(), 0), (logits[0], tokens, 0), (logits[:0], tokens[:0], 0)):
        with pytest.raises(RuntimeError):
            llmops.token_logprobs(*a)


def test_rows_further_apart_than_32_bits():
    """strides that take later rows past 2^31 elements from the first, for rows of many runs and of one"""
    far = torch.zeros(2100, 1 << 20, device="cuda")  # 8.8 GB
    far[2050, 777] = 5.0
    far[2091, 4000] = 3.0
    for logits, V in ((far[None, ::41], 1 << 20), (far[None, ::41, :5000], 5000), (far[::41, None, :20001], 20001)):
        shape = logits.shape[:2]
        tokens = torch.full(shape, 777, device="cuda")
        for top in (0, 2):
            lp, ent, ids, lps = llmops.token_logprobs(logits, tokens, top)
            lp, ent, ids, lps = lp.flatten(), ent.flatten(), ids.reshape(52, top), lps.reshape(52, top)
            for row, z in ((49, 0.0), (50, 5.0), (51, 0.0)):  # (logits of 777; the last row has 3 elsewhere)
                highest = (0.0, 5.0, 3.0)[row - 49]
                log_s = math.log(V - 1 + math.exp(highest))
                # p * distance from the top: at most that distance
                assert abs(float(lp[row]) - (z - log_s)) <= (2 * highest + 42 + 14) * E
                p = math.exp(highest - log_s)
                want = log_s - p * highest
                assert abs(float(ent[row]) - want) <= (2 * highest + 42 + 14 + highest * (2 * highest + 43) + highest * (2 * highest + 42)) * E
            if top:
                assert ids[49].tolist() == [0, 1] and ids[50].tolist() == [777, 0] and ids[51].tolist() == [4000, 0]
                assert abs(float(lps[50, 0] - lp[50])) == 0.0
