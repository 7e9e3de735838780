"""A cache in 4 bits through LlamaDecoder: turns, steps with drafted tokens, a beginning in common, scores.  End to end two evaluations drift by the 8-bit
rounding of activations (test_decode_gpu.py says why): logits are compared at its 5e-2 against the same model whose attention is
evaluated plainly over what the cache stands for; what must be the same bits is compared as such."""
import math

import pytest
import torch

import llmops
from conftest import max_rel_err
from llmops.decode import LlamaDecoder
from llmops.opset import Q4Cache

pytestmark = pytest.mark.gpu

CFG = dict(layer_num=2, head_num=2, head_size=128, hidden_size=256, intermediate_size=512, vocab_size=320, rms_norm_eps=1e-5, rope_base=10000.0)


def _ids(seed, *shape):
    return torch.randint(0, CFG["vocab_size"], shape, generator=torch.Generator().manual_seed(seed)).cuda()


class PlainCache(Q4Cache):
    """the same cache, attention evaluated in 64 bits over what it stands for"""

    def attend(self, q, k, v, inv_freq, layer_id, q_lens=None):
        llmops.cache_write_q4(k, v, self.cache, self.lengths, layer_id, inv_freq=inv_freq, q_lens=q_lens)
        K, V = self.read(dtype=torch.float32)[2 * layer_id:2 * layer_id + 2].double()
        B, L, width = q.shape
        row = self.lengths[:, None] + torch.arange(L, device="cuda")
        angle = row[..., None].double() * inv_freq.double()
        lo, hi = q.double().reshape(B, L, -1, 128).chunk(2, dim=-1)
        cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]
        x = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1).transpose(1, 2).contiguous()
        s = torch.matmul(x, K.transpose(2, 3).contiguous()) / math.sqrt(128)
        s = s.masked_fill((torch.arange(self.max_kv_len, device="cuda") > row[..., None])[:, None], -math.inf)
        out = torch.matmul(torch.softmax(s, dim=-1), V).transpose(1, 2).reshape(B, L, width)
        live = torch.arange(L, device="cuda") < (q_lens[:, None] if q_lens is not None else L)
        return torch.where(live[..., None], out, 0.0).float()


@pytest.mark.parametrize("plan", ["fused", "reference"])
@pytest.mark.parametrize("P", [0, 21])
def test_turns_and_tokens(plan, P):
    model = LlamaDecoder(CFG, seed=3, plan=plan)
    prefix = model.read_prefix(_ids(1, 1, P), torch.float16) if P else None
    cache = model.request_cache(3, 60, prefix, bits=4)
    assert isinstance(cache, Q4Cache) and cache.lengths.tolist() == [P] * 3 and cache.size() == 4 * 3 * 2 * (60 + P) * 80
    plain = PlainCache(CFG, 3, 60 + P)
    if P:
        plain.begin(prefix)
    n = torch.tensor([40, 2, 17], dtype=torch.int32).cuda()
    for step in range(5):
        ids, lens = (_ids(2, 3, 40), n) if step == 0 else (_ids(10 + step, 3, 1), None)
        a, b = model.forward_requests(ids, cache, lens), model.forward_requests(ids, plain, lens)
        for s in range(3):
            t = int(n[s]) if step == 0 else 1
            assert max_rel_err(a[s, :t].cpu().numpy(), b[s, :t].cpu().numpy()) <= 5e-2
        plain.cache.copy_(cache.cache)  # (codes that flip would drift apart)
        cache.keep(lens if lens is not None else 1), plain.keep(lens if lens is not None else 1)
    assert cache.lengths.tolist() == [P + 44, P + 6, P + 21]


def test_a_beginning_in_common():
    model = LlamaDecoder(CFG, seed=5)
    prefix = model.read_prefix(_ids(1, 1, 30))
    cache = model.request_cache(3, 10, prefix, bits=4)
    held = cache.read(30, dtype=torch.float32)
    assert torch.equal(held[:, :1].expand(-1, 3, -1, -1, -1), held)
    # within a step of every group of 32: a fifteenth of its range, and two units of the group's largest value's 1016th
    off, groups = (held[:, :1] - prefix).abs().unflatten(-1, (4, 32)), prefix.unflatten(-1, (4, 32))
    step = (groups.amax(-1) - groups.amin(-1)) / 15 + groups.abs().amax(-1) / 508
    assert (off.amax(-1) <= step).all()
    model.forward_requests(_ids(2, 3, 4), cache)
    cache.keep(4)
    cache.forget(1)
    cache.forget(2, 3)
    assert cache.lengths.tolist() == [34, 30, 33] and torch.equal(cache.read(30, dtype=torch.float32), held)
    # what was read back serves as a prefix in full width
    full = model.request_cache(2, 8, cache.read(30)[:, :1].contiguous())
    x = _ids(3, 2, 5)
    a = model.forward_requests(x, full)
    cache.begin(cache.read(30)[:, :1].contiguous())
    b = model.forward_requests(torch.cat((x, x[:1])), cache)
    # (its own five rows are in 4 bits, of 35)
    assert max_rel_err(b[:2].cpu().numpy(), a.cpu().numpy()) <= 0.2
    for bad in (lambda: cache.begin(prefix[:2]), lambda: cache.begin(prefix, 31), lambda: cache.begin(prefix[..., :64]), lambda: model.request_cache(1, 8, bits=3),
                lambda: model.request_cache(1, 8, dtype=torch.float16, bits=4), lambda: Q4Cache(dict(CFG, head_size=64), 1, 8), lambda: cache.forget(0, 11)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("K", [0, 3])
def test_steps_with_drafts_captured(K):
    """one graph serves following steps, with alternatives beside the tokens: the same as step by step"""
    model = LlamaDecoder(CFG, seed=6)
    prefix = model.read_prefix(_ids(1, 1, 9))
    caches = [model.request_cache(3, 16, prefix, bits=4) for _ in range(2)]
    tokens, uniforms = _ids(2, 3), torch.rand(3, K + 1, generator=torch.Generator().manual_seed(1)).cuda()
    drafts = _ids(3, 3, K)

    def step(cache):
        return model.step_requests(tokens, cache, uniforms, drafts if K else None, top=4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])  # (workspaces of this stream)
        caches[0].lengths.fill_(9)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            result, accepted, (logprobs, entropy, top, top_logprobs) = step(caches[0])
    caches[0].lengths.fill_(9)
    for i in range(6):
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        r, n, scores = step(caches[1])
        assert torch.equal(r, result) and torch.equal(n, accepted) and torch.equal(caches[0].lengths, caches[1].lengths)
        assert all(torch.equal(a, b) for a, b in zip((logprobs, entropy, top, top_logprobs), scores))
        assert logprobs.shape == (3, K + 1) and top.shape == (3, K + 1, 4) and (logprobs[result < 0] == 0).all() and (logprobs[result >= 0] < 0).all()
        tokens.copy_(r.gather(1, n[:, None].long())[:, 0].clamp(min=0))
        drafts.copy_(_ids(20 + i, 3, K)), uniforms.copy_(torch.rand(3, K + 1, generator=torch.Generator().manual_seed(50 + i)))
    assert (caches[0].lengths <= 25).all()


@pytest.mark.parametrize("bits", [None, 4])
def test_scores(bits):
    model = LlamaDecoder(CFG, seed=7)
    ids, n = _ids(4, 3, 30), torch.tensor([30, 11, 1], dtype=torch.int32).cuda()
    caches = [model.request_cache(3, 32, bits=bits) for _ in range(2)]
    lp, ent, top, top_lp = model.score_requests(ids, caches[0], n, top=5)
    logits = model.forward_requests(ids, caches[1], n).double()
    want = torch.log_softmax(logits[:, :-1], dim=-1)
    live = torch.arange(1, 30, device="cuda") < n[:, None]
    assert lp.shape == ent.shape == (3, 29) and top.shape == top_lp.shape == (3, 29, 5)
    # (tolerances: test_token_logprobs_gpu.py; logits here are within 20 of their top, 42 + 2 * 20 roundings)
    assert (lp - torch.where(live, want.gather(-1, ids[:, 1:, None])[..., 0], 0.0)).abs().max() <= 100 * 2.0 ** -24
    assert (top_lp - want.gather(-1, top)).abs().max() <= 100 * 2.0 ** -24
    assert torch.equal(top[..., 0], logits[:, :-1].argmax(-1))
    assert model.score_requests(ids, caches[0])[2].shape == (3, 29, 0)
    assert model.score_requests(_ids(5, 3, 1), caches[0], top=2)[3].shape == (3, 0, 2)


@pytest.mark.parametrize("bits", [None, 4])
def test_texts_that_do_not_fit(bits):
    model = LlamaDecoder(CFG, seed=8)
    ids = _ids(6, 3, 20)
    cache, wide = model.request_cache(3, 24, bits=bits), model.request_cache(3, 60, bits=bits)
    for c in (cache, wide):
        c.lengths.copy_(torch.tensor([0, 12, 24], dtype=torch.int32))
    lp, want = model.score_requests(ids, cache)[0], model.score_requests(ids, wide)[0]
    assert (lp[0] < 0).all() and (lp[0] - want[0]).abs().max() <= 5e-2 * want.abs().max()
    # rows 12 .. 23 are left for 12 tokens, the last of which says what the next one is worth
    # (caches of two capacities may add in different orders: codes of activations may flip, as above)
    assert (lp[1, :12] < 0).all() and (lp[1, 12:] == 0).all() and (lp[1, :12] - want[1, :12]).abs().max() <= 5e-2 * want.abs().max()
    assert (lp[2] == 0).all()


def test_what_is_refused_changes_nothing():
    model = LlamaDecoder(CFG, seed=9)
    prefix = model.read_prefix(_ids(1, 1, 5), torch.float16)
    cache = model.request_cache(2, 20, prefix, bits=4)
    tokens, uniforms = _ids(2, 2), torch.full((2, 1), 0.5, device="cuda")
    for top in (65, -1, CFG["vocab_size"] + 1):
        with pytest.raises(RuntimeError):
            model.step_requests(tokens, cache, uniforms, top=top)
    for length in (-1, 21):
        with pytest.raises(ValueError):
            cache.forget(0, length)
    for full in (prefix.bfloat16(), prefix.cpu(), prefix[:2], prefix[0], prefix.expand(-1, 2, -1, -1, -1)):
        with pytest.raises(ValueError):
            cache.begin(full)
    with pytest.raises(ValueError):
        cache.begin(prefix, 6)
    assert cache.lengths.tolist() == [5, 5] and cache.begun == 5
    cache.forget(1, 3)
    assert cache.lengths.tolist() == [5, 8]


@pytest.mark.parametrize("plan", ["fused", "reference"])
@pytest.mark.parametrize("bits", [None, 4])
def test_texts_padded_with_anything(bits, plan):
    """what lies behind a text's end has no effect on it: ids that are no tokens give the bits that tokens give"""
    model = LlamaDecoder(CFG, seed=10, plan=plan)
    n = torch.tensor([20, 7, 1], dtype=torch.int32).cuda()
    ids = _ids(7, 3, 20)
    behind = torch.arange(20, device="cuda") >= n[:, None]
    want = model.score_requests(ids, model.request_cache(3, 32, bits=bits), n, top=3)
    for pad in (-1, -100, CFG["vocab_size"], 1 << 40):
        got = model.score_requests(ids.masked_fill(behind, pad), model.request_cache(3, 32, bits=bits), n, top=3)
        live = ~behind[:, 1:]
        assert torch.equal(got[0], want[0])
        assert all(torch.equal(a[live], b[live]) for a, b in zip(got[1:], want[1:]))
        logits = model.forward_requests(ids.masked_fill(behind, pad), model.request_cache(3, 32, bits=bits), n)
        assert logits.isfinite().all()


def test_a_beginning_that_is_refused_changes_nothing():
    model = LlamaDecoder(CFG, seed=11)
    prefix = model.read_prefix(_ids(1, 1, 6))
    cache = model.request_cache(2, 20, prefix, bits=4)
    cache.keep(3)
    held = cache.cache.clone()
    wide = torch.zeros(4, 1, 2, 6, 256, device="cuda")
    flat = torch.zeros(prefix.numel() + 8192, device="cuda")
    strides = prefix.stride()
    inside = cache.cache.view(torch.float32).flatten()
    for full in (wide[..., ::2],                                                        # rows that are not dense
                 wide[..., 1:129],                                                      # an address between 16 bytes
                 flat[2:2 + prefix.numel()].view(prefix.shape),                         # ..
                 flat.as_strided(prefix.shape, (strides[0] + 2,) + strides[1:]),        # only later layers are
                 flat.as_strided(prefix.shape, strides[:2] + (strides[2] + 1,) + strides[3:]), flat.as_strided(prefix.shape, strides[:3] + (130, 1)),
                 flat.half().as_strided(prefix.shape, strides[:3] + (132, 1)),
                 inside.as_strided(prefix.shape, (0, 0, 0, 128, 1), inside.numel() - 6 * 128)):   # the cache's own memory
        with pytest.raises(ValueError):
            cache.begin(full)
        assert cache.begun == 6 and cache.lengths.tolist() == [9, 9] and torch.equal(cache.cache, held)
    # strides of dims of one element, and rows that lie apart, are none of the refused
    roomy = torch.zeros(4, 3, 2, 9, 128, device="cuda")[:, 1:2]
    roomy[:, :, :, :6] = prefix
    cache.begin(roomy, 6)
    assert torch.equal(cache.cache[..., :6, :], held[..., :6, :]) and cache.lengths.tolist() == [6, 6]
    cache.begin(prefix.as_strided(prefix.shape, (strides[0], 1) + strides[2:]), 6)
    assert torch.equal(cache.cache[..., :6, :], held[..., :6, :])
    cache.begin(flat.as_strided(prefix.shape, strides[:3] + (130, 1)), 1)
    assert cache.begun == 1 and cache.lengths.tolist() == [1, 1] and not cache.read(1).any()
    cache.begin(prefix, 0)
    assert cache.begun == 0 and cache.lengths.tolist() == [0, 0]


def test_tokens_taken_back_end_at_the_beginning():
    model = LlamaDecoder(CFG, seed=12)
    prefix = model.read_prefix(_ids(1, 1, 9))
    cache = model.request_cache(3, 16, prefix, bits=4)
    tokens = torch.tensor([5, 0, 16], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            cache.keep(tokens)

    def replay():
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()

    cache.keep(tokens)
    assert cache.lengths.tolist() == [14, 9, 25]
    cache.keep(-7)
    assert cache.lengths.tolist() == [9, 9, 18]
    cache.keep(torch.tensor([-1, 3, -100], dtype=torch.int32, device="cuda"))
    assert cache.lengths.tolist() == [9, 12, 9]
    cache.keep(40)
    assert cache.lengths.tolist() == [25, 25, 25]
    # a captured step, behind other beginnings than the one that it was captured with
    for rows in (9, 4, 0, 7):
        cache.begin(prefix, rows)
        replay()
        assert cache.lengths.tolist() == [rows + 5, rows, rows + 16]
        tokens.neg_(), replay()
        assert cache.lengths.tolist() == [rows] * 3
        tokens.neg_()
    assert cache.begun == 7
