"""Several requests in step through LlamaDecoder: shared prefix, adapters, drafted tokens together, against the calls that serve one
chat.  End to end two evaluations drift by the 8-bit rounding of activations (test_decode_gpu.py says why): logits are compared at its
5e-2, and what must be the same bits is compared as such."""
import numpy as np
import pytest
import torch

import llmops
from conftest import max_rel_err
from llmops.decode import LlamaDecoder
from llmops.opset import LoraAdapters, PrefixCache

pytestmark = pytest.mark.gpu

CFG = dict(layer_num=2, head_num=2, head_size=128, hidden_size=256, intermediate_size=512, vocab_size=320, rms_norm_eps=1e-5, rope_base=10000.0)


def _ids(seed, *shape):
    return torch.randint(0, CFG["vocab_size"], shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _adapters(seed, count=2, names=LlamaDecoder.PROJECTIONS, size=0.05):
    g = torch.Generator().manual_seed(seed)
    H, F = CFG["hidden_size"], CFG["intermediate_size"]
    width = {"gate_proj": (H, F), "up_proj": (H, F), "down_proj": (F, H)}
    layers = []
    for _ in range(CFG["layer_num"]):
        layer = {}
        for n in names:
            K, N = width.get(n, (H, H))
            layer[n] = [(torch.randn(r, K, generator=g) * size, torch.randn(N, r, generator=g) * size, 0.5 + i) for i, r in enumerate((4, 9, 16)[:count])]
        layers.append(layer)
    return layers


def _alone(model, ids):
    """logits of one sequence from nothing, through the calls for one chat"""
    cache = torch.zeros(2 * CFG["layer_num"], 1, CFG["head_num"], ids.shape[1], CFG["head_size"]).cuda()
    return model.forward(ids, cache, torch.arange(ids.shape[1], dtype=torch.int32).cuda(), 0)


@pytest.mark.parametrize("plan", ["fused", "reference"])
@pytest.mark.parametrize("group,half", [(128, False), (32, True)])
@pytest.mark.parametrize("P", [0, 21])
def test_turns_behind_a_prefix(plan, group, half, P):
    """ragged turns, then single tokens: the same logits as each sequence alone from its first token on"""
    model = LlamaDecoder(CFG, group_k=group, seed=3, plan=plan)
    dtype = torch.float16 if half else torch.float32
    shared = _ids(1, 1, P) if P else None
    cache = model.request_cache(3, 24, model.read_prefix(shared, dtype) if P else None, dtype)
    turns, n = _ids(2, 3, 7), torch.tensor([7, 2, 5], dtype=torch.int32).cuda()
    said = [turns[b, :int(n[b])] for b in range(3)]
    logits = model.forward_requests(turns, cache, n)
    cache.keep(n)
    steps = [[logits[b, :int(n[b])]] for b in range(3)]
    for step in range(3):
        more = _ids(10 + step, 3, 1)
        logits = model.forward_requests(more, cache)
        cache.keep(1)
        for b in range(3):
            said[b] = torch.cat((said[b], more[b]))
            steps[b].append(logits[b])
    assert cache.lengths.tolist() == [10, 5, 8]
    for b in range(3):
        want = _alone(model, torch.cat((shared[0], said[b]))[None] if P else said[b][None])[0, P:]
        assert max_rel_err(torch.cat(steps[b]).cpu().numpy(), want.cpu().numpy()) <= 5e-2


def test_a_prefix_is_shared_and_left_alone():
    model = LlamaDecoder(CFG, seed=3)
    prefix = model.read_prefix(_ids(1, 1, 12))
    before = prefix.clone()
    a, b = model.request_cache(2, 8, prefix), model.request_cache(1, 8, prefix)
    x = _ids(2, 2, 4)
    la, lb = model.forward_requests(x, a), model.forward_requests(x[1:], b)
    assert torch.equal(prefix, before) and a.size() == b.size() + b.cache.numel() * 4
    assert max_rel_err(la[1:].cpu().numpy(), lb.cpu().numpy()) <= 5e-2
    a.keep(4)
    a.forget(1)
    assert a.lengths.tolist() == [4, 0]
    again = model.forward_requests(x, a, q_lens=torch.tensor([0, 4], dtype=torch.int32).cuda())
    assert max_rel_err(again[1].cpu().numpy(), la[1].cpu().numpy()) <= 5e-2
    with pytest.raises(ValueError):
        PrefixCache(CFG, 1, 8, prefix, 13)
    with pytest.raises(ValueError):
        PrefixCache(CFG, 1, 8, prefix, 3, dtype=torch.float16)


@pytest.mark.parametrize("plan", ["fused", "reference"])
def test_adapters_change_their_own_requests_only(plan):
    model = LlamaDecoder(CFG, seed=4, plan=plan)
    x = _ids(5, 4, 3)

    def logits(numbers):
        cache = model.request_cache(4, 8)
        return model.forward_requests(x, cache, adapters=None if numbers is None else torch.tensor(numbers, dtype=torch.int32).cuda())

    with pytest.raises(RuntimeError, match="no adapters"):
        logits([0, 0, 0, 0])
    model.set_adapters(_adapters(1))
    none, two, three = logits([-1] * 4), logits([-1, 1, -1, 0]), logits([0, 1, -1, 0])
    plain = logits(None)  # (the norms ride in the products' launches: another order of sums)
    assert max_rel_err(none.cpu().numpy(), plain.cpu().numpy()) <= 5e-2
    assert torch.equal(two[[0, 2]], none[[0, 2]]) and torch.equal(three[1:], two[1:])
    for b in (1, 3):
        assert (two[b] - none[b]).abs().max() > 0.02 * none[b].abs().max()
    model.set_adapters(_adapters(1, size=0.0))
    assert torch.equal(logits([0, 1, 1, 0]), none)
    model.set_adapters(_adapters(1, names=("o_proj", "v_proj")))
    some = logits([-1, 1, -1, 0])
    assert torch.equal(some[[0, 2]], logits([-1] * 4)[[0, 2]])
    model.set_adapters(None)
    with pytest.raises(RuntimeError, match="no adapters"):
        logits([0, 0, 0, 0])
    for bad in ([{}], [{"q": []}, {}], [{"q_proj": [None]}, {"v_proj": [None, None]}]):
        with pytest.raises(ValueError):
            model.set_adapters(bad)
    with pytest.raises(ValueError):
        LoraAdapters([(torch.zeros(2, 8), torch.zeros(8, 3), 1.0)])


def test_an_adapter_is_what_the_projection_adds():
    """o_proj's adapter alone in a model of one layer: the layer's input to the MLP is off by scale * (attn A^T) B^T"""
    from llmops import opset
    A, B = torch.randn(5, 256, generator=torch.Generator().manual_seed(1)), torch.randn(256, 5, generator=torch.Generator().manual_seed(2))
    lora = opset.LoraAdapters([None, (A, B, 0.25)], dtype=torch.float32)
    assert lora.A.shape == (2, 8, 256)
    x, y = torch.randn(3, 2, 256).cuda(), torch.randn(3, 2, 256).cuda()
    want = y.double()
    want[1] += 0.25 * (x[1].double() @ A.double().T.cuda() @ B.double().T.cuda())
    got = lora(y, x, torch.tensor([0, 1, -1], dtype=torch.int32).cuda())
    assert got is y and (got.double() - want).norm() <= 4e-6 * want.norm()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("with_probs", [False, True])
def test_steps_with_drafts(half, with_probs):
    """answers are verify_drafts' on the model's logits, and what is kept serves the following steps as if it had come token by token"""
    model = LlamaDecoder(CFG, seed=6)
    model.set_adapters(_adapters(3))
    numbers = torch.tensor([0, -1, 1], dtype=torch.int32).cuda()
    dtype = torch.float16 if half else torch.float32
    prefix = model.read_prefix(_ids(1, 1, 30), dtype)
    cache, plain = model.request_cache(3, 40, prefix), model.request_cache(3, 40, prefix)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens, said = _ids(2, 3), [[], [], []]
    lens = torch.tensor([4, 1, 3], dtype=torch.int32).cuda()
    for step in range(4):
        # drafts: half of the time the model's own choice (from the caches as they are), so that some are accepted
        probs = torch.softmax(2 * torch.randn(3, 4, CFG["vocab_size"], generator=g, device="cuda"), -1) if with_probs else None
        drafts = torch.randint(0, CFG["vocab_size"], (3, 4), generator=g, device="cuda")
        own = model.forward_requests(torch.cat((tokens[:, None], drafts), 1), cache, lens + 1, numbers).argmax(-1)[:, :1]
        drafts[:, :1] = torch.where(torch.rand(3, 1, generator=g, device="cuda") < 0.7, own, drafts[:, :1])
        uniforms = torch.rand(3, 5, generator=g, device="cuda")
        before = cache.lengths.clone()
        logits = model.forward_requests(torch.cat((tokens[:, None], drafts), 1), cache, lens + 1, numbers)
        want = llmops.verify_drafts(logits, drafts, uniforms, draft_probs=probs, temperature=0.5, draft_lens=lens)
        result, accepted = model.step_requests(tokens, cache, uniforms, drafts, probs, lens, 0.5, numbers)
        assert torch.equal(result, want[0]) and torch.equal(accepted, want[1])
        assert torch.equal(cache.lengths, before + accepted + 1)
        for b in range(3):
            for t in [int(tokens[b])] + result[b, :int(accepted[b])].tolist():
                said[b].append(t)
        tokens = result.gather(1, accepted[:, None].long())[:, 0]
        assert (tokens >= 0).all()
    # the same tokens one by one
    for b in range(3):
        assert int(cache.lengths[b]) == len(said[b])
    longest = max(map(len, said))
    for i in range(longest):
        ids = torch.tensor([[s[i] if i < len(s) else 0] for s in said]).cuda()
        n = torch.tensor([int(i < len(s)) for s in said], dtype=torch.int32).cuda()
        model.forward_requests(ids, plain, n, numbers)
        plain.keep(n)
    assert torch.equal(plain.lengths, cache.lengths)
    got = model.forward_requests(tokens[:, None], cache, adapters=numbers)
    want = model.forward_requests(tokens[:, None], plain, adapters=numbers)
    assert max_rel_err(got.cpu().numpy(), want.cpu().numpy()) <= 5e-2
    for b in range(3):
        n = len(said[b])
        a, c = cache.cache[:, b, :, :n].float(), plain.cache[:, b, :, :n].float()
        assert (a - c).abs().max() <= 5e-2 * c.abs().max()


def test_step_without_drafts_and_tokens_outside():
    model = LlamaDecoder(CFG, seed=6)
    cache = model.request_cache(2, 9)
    result, accepted = model.step_requests(_ids(1, 2), cache, torch.rand(2, 1).cuda(), temperature=0.0)
    assert result.shape == (2, 1) and accepted.tolist() == [0, 0] and cache.lengths.tolist() == [1, 1]
    result, accepted = model.step_requests(result[:, 0], cache, torch.rand(2, 3).cuda(), torch.tensor([[-1, 5], [1 << 40, -7]]).cuda())
    assert accepted.tolist() == [0, 0] and cache.lengths.tolist() == [2, 2] and ((0 <= result[:, 0]) & (result[:, 0] < CFG["vocab_size"])).all()


def test_a_captured_step_serves_the_following_ones():
    model = LlamaDecoder(CFG, seed=8)
    model.set_adapters(_adapters(2, count=3))
    prefix = model.read_prefix(_ids(1, 1, 17))
    numbers = torch.tensor([2, 0, -1, 1], dtype=torch.int32).cuda()
    tokens, drafts, lens = _ids(2, 4), _ids(3, 4, 2), torch.tensor([2, 1, 0, 2], dtype=torch.int32).cuda()
    uniforms = torch.rand(4, 3, generator=torch.Generator().manual_seed(1)).cuda()
    cache, eager = model.request_cache(4, 32, prefix), model.request_cache(4, 32, prefix)
    args = dict(uniforms=uniforms, drafts=drafts, draft_lens=lens, temperature=0.8, adapters=numbers)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        model.step_requests(tokens, model.request_cache(4, 32, prefix), **args)  # (workspaces of this stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            result, accepted = model.step_requests(tokens, cache, **args)
    torch.cuda.synchronize()
    for step in range(5):
        want = model.step_requests(tokens, eager, **args)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(result, want[0]) and torch.equal(accepted, want[1]) and torch.equal(cache.lengths, eager.lengths)
        assert torch.equal(cache.cache, eager.cache)
        tokens.copy_(result.gather(1, accepted[:, None].long())[:, 0])
        drafts.copy_(_ids(20 + step, 4, 2))
        uniforms.copy_((uniforms * 3.7) % 1.0)
        torch.cuda.synchronize()


@pytest.mark.parametrize("given", [None, [2, 4, 4, 1]])
def test_a_step_at_the_end_of_the_cache(given):
    """drafts that no longer fit are not checked, and a sequence without room for its token gives none; the others are as they are"""
    model = LlamaDecoder(CFG, seed=9)
    cache, other = (model.request_cache(4, 9, model.read_prefix(_ids(1, 1, 11))) for _ in range(2))
    said = torch.tensor([0, 5, 8, 9], dtype=torch.int32).cuda()
    model.forward_requests(_ids(2, 4, 9), cache, said)
    cache.keep(said)
    other.cache.copy_(cache.cache), other.lengths.copy_(cache.lengths)
    tokens, drafts = _ids(3, 4), _ids(4, 4, 4)
    uniforms = torch.zeros(4, 5).cuda()  # (every draft that is checked is accepted)
    uniforms[:, 4] = 0.4
    lens = None if given is None else torch.tensor(given, dtype=torch.int32).cuda()
    fit = [4, 3, 0, 0] if given is None else [2, 3, 0, 0]
    result, accepted = model.step_requests(tokens, cache, uniforms, drafts, draft_lens=lens)
    assert accepted.tolist() == fit and cache.lengths.tolist() == [fit[0] + 1, 9, 9, 9]
    assert (result[3] == -1).all()
    for b in range(3):
        n = fit[b]
        assert torch.equal(result[b, :n], drafts[b, :n]) and 0 <= int(result[b, n]) < CFG["vocab_size"] and (result[b, n + 1:] == -1).all()
    want, _ = model.step_requests(tokens, other, uniforms, drafts, draft_lens=torch.tensor(fit, dtype=torch.int32).cuda())
    assert torch.equal(result, want) and torch.equal(cache.cache, other.cache)
    # a token that was not given goes nowhere
    before = cache.cache.clone()
    result, accepted = model.step_requests(result.gather(1, accepted[:, None].long())[:, 0], cache, uniforms[:, :1].contiguous())
    assert (result[1:] == -1).all() and accepted.tolist() == [0] * 4 and int(result[0, 0]) >= 0 and cache.lengths.tolist() == [fit[0] + 2, 9, 9, 9]
    assert torch.equal(cache.cache[:, 1:], before[:, 1:])
