"""lora_add against the formula in 64 bits.

Tolerances.  Products are formed of exact pieces, what is dropped is below 2^-22 of a product, and sums are fp32: a value of x A^T (K
products ~N(0, 1) / sqrt(K)) is off by about 1e-6 of its size at most, and so the delta: 4e-6 of the delta's 2-norm, and one rounding of y
(2^-24) beside it; the largest of some 10^6 values by ten times that."""
import math

import pytest
import torch

import llmops

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _case(B, M, N, K, R, n, dtype, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    x, y = torch.randn(B, M, K, generator=g), torch.randn(B, M, N, generator=g)
    A = (torch.randn(n, R, K, generator=g) / math.sqrt(K)).to(TYPES[dtype])
    W = (torch.randn(n, N, R, generator=g) / math.sqrt(R)).to(TYPES[dtype])
    scales = torch.rand(n, generator=g) + 0.5
    ids = torch.randint(-1, n, (B,), generator=g) if ids is None else torch.as_tensor(ids)
    return y, x, A, W, ids.to(torch.int32), scales


def _delta(x, A, W, ids, scales):
    d = torch.zeros(*x.shape[:2], W.shape[1], dtype=torch.float64)
    for b, a in enumerate(ids.tolist()):
        if 0 <= a < A.shape[0]:
            d[b] = scales[a].double() * (x[b].double() @ A[a].double().T @ W[a].double().T)
    return d


def _check(got, y, d):
    got = got.cpu().double()
    err = got - (y.double() + d)
    none = (d == 0).all(-1)
    assert torch.equal(got[none], y.double()[none])
    assert err.norm() <= 4e-6 * d.norm() + 2.0 ** -24 * got.norm()
    assert err.abs().max() <= 4e-5 * d.abs().max() + 2.0 ** -24 * got.abs().max()


def _run(case, **kw):
    return llmops.lora_add(*(t.cuda() for t in case), **kw)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,M,N,K,R,n", [
    (1, 1, 64, 64, 8, 1), (1, 1, 1, 1, 1, 1), (3, 1, 100, 130, 4, 2), (16, 1, 256, 512, 16, 16), (17, 1, 300, 257, 10, 5), (5, 7, 130, 96, 33, 3),
    (2, 40, 512, 1000, 64, 2), (33, 2, 77, 4096, 24, 40), (1, 100, 1030, 264, 130, 1), (4, 3, 4, 8, 300, 3), (6, 16, 640, 2048, 16, 6), (1, 2, 4096, 11008, 8, 1),
])
def test_against_64_bits(B, M, N, K, R, n, dtype):
    case = _case(B, M, N, K, R, n, dtype, seed=B + 10 * M)
    _check(_run(case), case[0], _delta(*case[1:]))


# 32 tokens to a tile: tiles of one sequence and of several, ranks past 128, rows and ranks shorter than eight, sizes that fill nothing
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,M,N,K,R,n", [(4, 100, 260, 520, 16, 3), (350, 1, 130, 264, 16, 5), (2, 200, 1030, 96, 64, 2), (5, 70, 77, 4, 3, 2), (1, 330, 100, 2049, 140, 1),
                                         (66, 5, 640, 1000, 40, 7), (11, 33, 65, 31, 5, 4)])
def test_many_tokens(B, M, N, K, R, n, dtype):
    case = _case(B, M, N, K, R, n, dtype, seed=B + 10 * M)
    _check(_run(case), case[0], _delta(*case[1:]))


@pytest.mark.parametrize("ids", [[-1] * 6, [0] * 6, [2, 1, 0, 2, 1, 0], [-1, 3, 2, 99, -7, 0]])
def test_which_adapter(ids):
    case = _case(6, 5, 200, 320, 16, 3, "fp16", seed=1, ids=ids)
    _check(_run(case), case[0], _delta(*case[1:]))


def test_long_prompts_and_in_place():
    case = _case(3, 700, 520, 768, 32, 2, "bf16", seed=4, ids=[1, -1, 0])
    d = _delta(*case[1:])
    _check(_run(case), case[0], d)
    y = case[0].cuda()
    assert llmops.lora_add(y, *(t.cuda() for t in case[1:]), out=y) is y
    _check(y, case[0], d)


@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_columns_of_a_fused_projection(at):
    """y and x are columns of wider rows, at every alignment"""
    y, x, A, W, ids, scales = _case(4, 3, 96, 160, 16, 3, "fp16", seed=at)
    wide_y, wide_x = torch.randn(4, 3, 300).cuda(), torch.randn(4, 3, 333).cuda()
    wide_y[..., at:at + 96], wide_x[..., at:at + 160] = y.cuda(), x.cuda()
    before = wide_y.clone()
    part = wide_y[..., at:at + 96]
    out = llmops.lora_add(part, wide_x[..., at:at + 160], A.cuda(), W.cuda(), ids.cuda(), scales.cuda(), out=part)
    _check(out, y, _delta(x, A, W, ids, scales))
    before[..., at:at + 96] = out
    assert torch.equal(wide_y, before)


def test_numbers_stay_with_their_requests():
    """an adapter that holds NaN or infinities, or a request that does, changes nothing for the others of its tile"""
    y, x, A, W, ids, scales = _case(12, 1, 128, 256, 16, 4, "fp32", seed=3, ids=[0, 1, 2, 3, -1, 0, 1, 2, 3, -1, 0, 1])
    want = _run((y, x, A, W, ids, scales))
    A[1, 3, 5], W[2, 7, 2], x[5, 0, 9], x[4, 0, 3] = math.nan, math.inf, math.inf, math.nan
    got = _run((y, x, A, W, ids, scales))
    clean = [0, 3, 4, 8, 9, 10]
    assert torch.equal(got[clean], want[clean])
    assert torch.isnan(got[[1, 6, 11]]).all() and not torch.isfinite(got[[2, 7], :, 7]).any() and not torch.isfinite(got[5]).any()
    assert torch.isfinite(got[[2, 7]][..., :7]).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("xs,ws", [(1e-20, 1.0), (1e20, 1.0), (1e5, 1e-4), (3e-5, 100.0)])
def test_magnitudes(xs, ws, dtype):
    y, x, A, W, ids, scales = _case(4, 2, 64, 96, 16, 2, dtype, seed=2, ids=[0, 1, 0, 1])
    x, A, y = x * xs, (A.float() * ws).to(A.dtype), y * xs * ws
    _check(_run((y, x, A, W, ids, scales)), y, _delta(x, A, W, ids, scales))


def test_graph_and_streams():
    case = [t.cuda() for t in _case(9, 2, 320, 512, 16, 4, "bf16", seed=5)]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        llmops.lora_add(*case)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = llmops.lora_add(*case)
    torch.cuda.synchronize()
    for _ in range(4):
        case[4].copy_((case[4] + 2) % 5 - 1)  # (adapters change between replays)
        case[1].mul_(0.5)
        want = llmops.lora_add(*case)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals():
    y, x, A, W, ids, scales = (t.cuda() for t in _case(2, 2, 32, 48, 8, 2, "fp16", seed=1))
    llmops.lora_add(y, x, A, W, ids, scales)
    for args in ((y.cpu(), x, A, W, ids, scales), (y, x.half(), A, W, ids, scales), (y, x, A.float(), W, ids, scales), (y, x, A[:1], W, ids, scales),
                 (y, x, A, W, ids.long(), scales), (y, x, A, W, ids[:1], scales), (y, x, A, W, ids, scales[:1]), (y, x[:, :1], A, W, ids, scales),
                 (y, x, A.transpose(1, 2), W, ids, scales), (y, x, A, W[:, :16], ids, scales), (y, x, A.double(), W.double(), ids, scales), (y[0], x, A, W, ids, scales),
                 (y.transpose(1, 2), x, A, W, ids, scales), (y, x, A, W, ids.cpu(), scales)):
        with pytest.raises(RuntimeError):
            llmops.lora_add(*args)
    with pytest.raises(RuntimeError, match="rows apart"):
        llmops.lora_add(y, x, A, W, ids, scales, out=y[:1].expand(2, -1, -1))
    with pytest.raises(RuntimeError):
        llmops.lora_add(y, x, A, W, ids, scales, out=y[:, :1])
    for strides in ((32, 32, 1), (48, 32, 1), (32, 48, 1), (64, 31, 1), (31, 64, 1)):  # rows one in the other
        with pytest.raises(RuntimeError, match="rows apart"):
            llmops.lora_add(y, x, A, W, ids, scales, out=torch.empty(200, device="cuda").as_strided((2, 2, 32), strides))
    for strides in ((64, 32, 1), (32, 64, 1), (100, 40, 1)):
        out = torch.empty(200, device="cuda").as_strided((2, 2, 32), strides)
        assert torch.equal(llmops.lora_add(y, x, A, W, ids, scales, out=out), llmops.lora_add(y, x, A, W, ids, scales))


def test_offsets_past_32_bits():
    """the last of many sequences whose x is more than 2^32 values"""
    B, M, K, N = 1 << 10, 1 << 10, 4100, 32
    y, x1, A, W, _, scales = _case(1, M, N, K, 8, 1, "fp16", seed=13)
    x = torch.zeros(B, M, K, device="cuda")
    x[B - 1] = x1[0].cuda()
    ids = torch.zeros(B, dtype=torch.int32)
    out = llmops.lora_add(y.cuda().expand(B, M, N), x, A.cuda(), W.cuda(), ids.cuda(), scales.cuda())
    _check(out[B - 1:], y, _delta(x1, A, W, ids[:1], scales))
    assert torch.equal(out[:B - 1], y.cuda().expand(B - 1, M, N))


def test_x_y_and_out_beside_each_other_in_one_tensor():
    """columns of one wide tensor, and sequences between each other's: nothing lies over anything"""
    y, x, A, W, ids, scales = _case(4, 3, 96, 160, 16, 3, "fp16", seed=7)
    d = _delta(x, A, W, ids, scales)
    rest = [t.cuda() for t in (A, W, ids, scales)]
    for at_y, at_x, at_out in ((0, 96, 256), (0, 96, 0), (160, 0, 256), (256, 0, 160), (160, 0, 160)):
        wide = torch.randn(4, 3, 352).cuda()
        wide[..., at_y:at_y + 96], wide[..., at_x:at_x + 160] = y.cuda(), x.cuda()
        before = wide.clone()
        out = wide[..., at_out:at_out + 96]
        assert llmops.lora_add(wide[..., at_y:at_y + 96], wide[..., at_x:at_x + 160], *rest, out=out) is out
        _check(out, y, d)
        before[..., at_out:at_out + 96] = out
        assert torch.equal(wide, before)
    flat = torch.zeros(4, 3, 2, 160).cuda()  # out's rows between x's
    flat[:, :, 0] = x.cuda()
    _check(llmops.lora_add(y.cuda(), flat[:, :, 0], *rest, out=flat[:, :, 1, 64:]), y, d)


def test_outputs_over_inputs_are_refused():
    y, x, A, W, ids, scales = (t.cuda() for t in _case(2, 2, 32, 48, 8, 2, "fp16", seed=1))
    some = torch.zeros(2, 2, 100, device="cuda")
    for args in ((some[..., :32], x, some[..., 4:36]), (y, some[..., 10:58], some[..., 50:82]), (some[..., :32], x, some.flatten()[:128].view(2, 2, 32)),
                 (y, some[..., :48], some.flatten()[96:224].view(2, 2, 32)), (some[:1, :, :32].expand(2, -1, -1), x, some[..., :32])):
        before = some.clone()
        with pytest.raises(RuntimeError, match="apart"):
            llmops.lora_add(args[0], args[1], A, W, ids, scales, out=args[2])
        assert torch.equal(some, before)
