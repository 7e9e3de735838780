"""Rows of the 4-bit cache as they are written and read back, against the definition in 64 bits on the host: bytes have to be equal."""
import math

import numpy as np
import pytest
import torch

import llmops
import q4_reference as ref

pytestmark = pytest.mark.gpu


def _inv_freq(half=64):
    return 1.0 / (10000.0 ** (torch.arange(0, 2 * half, 2).float() / (2 * half)))


def _same(cache, want):
    got = cache.cpu().numpy()
    bad = np.argwhere(got != want)
    assert not len(bad), (len(bad), bad[:5])


@pytest.mark.parametrize("turn", [64, 32, 20, None])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("B,L,Hkv,maxlen", [(1, 1, 1, 1), (2, 1, 32, 40), (3, 17, 5, 33), (1, 130, 4, 200), (4, 16, 8, 16), (70, 2, 3, 9)])
def test_rows_as_written(B, L, Hkv, maxlen, dtype, turn):
    g = torch.Generator().manual_seed(B + L)
    k, v = (torch.randn(B, L, Hkv, 128, generator=g) * torch.randn(Hkv, 128, generator=g).exp() + torch.randn(Hkv, 128, generator=g) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    lengths = torch.randint(-2, maxlen + 2, (B,), generator=g, dtype=torch.int32)
    q_lens = torch.randint(-1, L + 2, (B,), generator=g, dtype=torch.int32)
    f = None if turn is None else _inv_freq(turn)
    for lens in (None, q_lens):
        cache = torch.randint(-128, 128, (4, B, Hkv, maxlen, 80), generator=g, dtype=torch.int8)  # (rows that are not written stay as they are)
        want = cache.numpy().copy()
        ref.write(want, k.numpy(), v.numpy(), 1, lengths, lens, None if f is None else f.numpy())
        dev = cache.cuda()
        llmops.cache_write_q4(k.cuda(), v.cuda().flatten(2), dev, lengths.cuda(), 1, inv_freq=None if f is None else f.cuda(), q_lens=None if lens is None else lens.cuda())
        _same(dev, want)


def test_far_positions():
    g = torch.Generator().manual_seed(1)
    maxlen = 1 << 20
    k, v = torch.randn(1, 9, 1, 128, generator=g), torch.randn(1, 9, 1, 128, generator=g)
    f = _inv_freq()
    f[0] = 1000.25
    dev = torch.zeros(2, 1, 1, maxlen, 80, dtype=torch.int8, device="cuda")
    llmops.cache_write_q4(k.cuda(), v.cuda(), dev, torch.tensor([maxlen - 9], dtype=torch.int32, device="cuda"), 0, inv_freq=f.cuda())
    pos = np.arange(maxlen - 9, maxlen)[:, None]
    want = np.stack((ref.quantise(ref.turned(k[0].double().numpy(), f.numpy(), pos)), ref.quantise(v[0].numpy())))[:, :, 0]
    _same(dev[:, 0, 0, -9:], want)
    assert not dev[:, 0, 0, :-9].any()


def _write_one(v, dtype=torch.float32):
    """rows [n, 128] as they come"""
    x = v.to(dtype).cuda()[None, :, None, :]
    cache = torch.zeros(2, 1, 1, v.shape[0], 80, dtype=torch.int8, device="cuda")
    llmops.cache_write_q4(x, x, cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 0)
    assert torch.equal(cache[0], cache[1])
    return cache


def test_borders_between_codes():
    # whole numbers and halves of the group's unit: values in the middle between two levels, which have to go to the even one
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-4064, 4065, (400, 128), generator=g).float() / 2
    x[:100] = (x[:100] / 64).round()
    x[100:200] = (x[100:200] / 500).round() / 2
    x[:, 0::32] = 2032.0  # (u = 1)
    x[200:, 1::32] = torch.randint(-2032, 2033, (200, 4), generator=g).float()
    x[::3] *= 2.0 ** -9
    _same(_write_one(x)[0, 0, 0], ref.quantise(x.numpy()))


@pytest.mark.parametrize("scale", [65024.0, 1.0, 2.0 ** -13, 2.0 ** -14, 2.0 ** -20, 2.0 ** -24, 2.0 ** -25, 2.0 ** -26, 1e-30, 1e-45, 0.0])
def test_magnitudes(scale):
    g = torch.Generator().manual_seed(3)
    x = (2 * torch.rand(64, 128, generator=g) - 1).double()
    x[:, 5] = 1.0
    x[:, 40] = -1.0
    x[20:, 64:96] = 0.0
    x[30:, 96:] = 0.37  # (all of a group equal)
    x = (x * scale).float()
    cache = _write_one(x)
    want = ref.quantise(x.numpy())
    _same(cache[0, 0, 0], want)
    back = llmops.cache_read_q4(cache, 64, dtype=torch.float32)[0, 0, 0].cpu().double().numpy()
    assert np.array_equal(back, ref.values(want))
    # a value is off by half a step at most, a step being a fifteenth of the group's range and less than 2 units more (the rounded ends, and up)
    t = x.double().numpy().reshape(64, 4, 32)
    most = np.abs(t).max(-1)
    step = (t.max(-1) - t.min(-1)) / 15 + 2 * np.maximum(most / 1016, 2.0 ** -24)
    assert (np.abs(back.reshape(64, 4, 32) - t) <= 0.5 * step[..., None] + np.maximum(most / 1016, 2.0 ** -24)[..., None]).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65025.0, -70000.0, 3e38])
def test_rows_that_halves_do_not_hold(bad):
    x = torch.randn(8, 128, generator=torch.Generator().manual_seed(4))
    for row in (1, 4, 7):
        x[row, 17 * row] = bad
    cache = _write_one(x)
    _same(cache[0, 0, 0], ref.quantise(x.numpy()))
    back = llmops.cache_read_q4(cache, 8)[0, 0, 0]
    assert back[[1, 4, 7]].isnan().all() and not back[[0, 2, 3, 5, 6]].isnan().any()
    # turned, too (what counts is the turned value: 65025 may have become less, and its neighbour more)
    f = _inv_freq().cuda()
    k = x.cuda()[None, :, None, :]
    llmops.cache_write_q4(k, k, cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 0, inv_freq=f)
    with np.errstate(invalid="ignore"):
        turned = ref.turned(x.double().numpy(), f.cpu().numpy(), np.arange(8))
    _same(cache[0, 0, 0], ref.quantise(turned))


def test_strides_and_shared_rows():
    g = torch.Generator().manual_seed(5)
    B, L, Hkv, maxlen = 3, 21, 4, 50
    full = torch.randn(2, 1, Hkv, 30, 128, generator=g).half()  # another cache's rows
    lengths = torch.tensor([0, 29, 40], dtype=torch.int32)
    wide = torch.randn(B, L, 3, Hkv * 128, generator=g)
    for k, v, f in ((full[0, :, :, 4:4 + L].transpose(1, 2).expand(B, -1, -1, -1), full[1, :, :, 4:4 + L].transpose(1, 2).expand(B, -1, -1, -1), None),
                    (full[0, :, :, 4:4 + L].transpose(1, 2).expand(B, -1, -1, -1), full[1, :, :, 4:4 + L].transpose(1, 2).expand(B, -1, -1, -1), _inv_freq()),
                    (wide[:, :, 1], wide[:, :, 2], _inv_freq()), (wide[:, :, 0], wide[:, :, 2], None)):
        want = np.zeros((2, B, Hkv, maxlen, 80), np.int8)
        ref.write(want, k.reshape(B, L, Hkv, 128).numpy(), v.reshape(B, L, Hkv, 128).numpy(), 0, lengths, None, None if f is None else f.numpy())
        dev = torch.zeros(2, B, Hkv, maxlen, 80, dtype=torch.int8, device="cuda")
        if k.dim() == 4:  # (the views themselves, on the device)
            src = full.cuda()
            kd, vd = (src[i, :, :, 4:4 + L].transpose(1, 2).expand(B, -1, -1, -1) for i in (0, 1))
        else:
            src = wide.cuda()
            kd, vd = src[:, :, 1 if f is not None else 0], src[:, :, 2]
        llmops.cache_write_q4(kd, vd, dev, lengths.cuda(), 0, inv_freq=None if f is None else f.cuda())
        _same(dev, want)


@pytest.mark.parametrize("B", [12, 13, 40])
def test_rows_that_many_sequences_share(B):
    g = torch.Generator().manual_seed(B)
    L, Hkv, maxlen = 50, 3, 70
    k, v, own = (torch.randn(n, L, Hkv, 128, generator=g).half() for n in (1, 1, B))
    lengths = torch.randint(-2, maxlen + 3, (B,), generator=g, dtype=torch.int32)
    q_lens = torch.randint(-1, L + 2, (B,), generator=g, dtype=torch.int32)
    kd, vd, ownd = k.cuda().expand(B, -1, -1, -1), v.cuda().expand(B, -1, -1, -1), own.cuda()
    for lens in (None, q_lens):
        for values, on in ((v.expand(B, -1, -1, -1), vd), (own, ownd)):  # (both in common; k alone)
            want = np.full((2, B, Hkv, maxlen, 80), 3, np.int8)
            ref.write(want, k.expand(B, -1, -1, -1).numpy(), values.numpy(), 0, lengths, lens, None)
            dev = torch.full((2, B, Hkv, maxlen, 80), 3, dtype=torch.int8, device="cuda")
            llmops.cache_write_q4(kd, on, dev, lengths.cuda(), 0, q_lens=None if lens is None else lens.cuda())
            _same(dev, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("planes,B,Hkv,maxlen,rows", [(2, 1, 1, 1, 1), (4, 3, 5, 33, 33), (2, 2, 32, 200, 7), (2, 67, 3, 20, 41)])
def test_read_back(planes, B, Hkv, maxlen, rows, dtype):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(planes, B, Hkv, maxlen, 128, generator=g) * 3
    cache = torch.from_numpy(ref.quantise(x.numpy()))
    full = ref.values(cache.numpy())
    starts = torch.randint(-3, maxlen + 2, (B,), generator=g, dtype=torch.int32)
    for first in (None, starts):
        want = np.zeros((planes, B, Hkv, rows, 128))
        for b in range(B):
            for r in range(rows):
                at = r + (0 if first is None else int(first[b]))
                if 0 <= at < maxlen:
                    want[:, b, :, r] = full[:, b, :, at]
        got = llmops.cache_read_q4(cache.cuda(), rows, starts=None if first is None else first.cuda(), dtype=dtype)
        assert got.dtype == dtype and np.array_equal(got.cpu().double().numpy(), want)
    assert llmops.cache_read_q4(cache.cuda(), 0).shape == (planes, B, Hkv, 0, 128)


def test_what_was_read_back_is_written_again():
    # halves of a cache in 4 bits, cut again: levels may lie closer, values stay within a step; and the bytes of a second round stand for the same
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(7))
    first = llmops.cache_read_q4(_write_one(x), 50)[0, 0, 0]
    again = llmops.cache_read_q4(_write_one(first.cpu(), torch.float16), 50)[0, 0, 0]
    assert torch.equal(first, again)


def test_offsets_past_32_bits():
    heads, maxlen = 60, 1 << 20  # 5 GB a plane
    cache = torch.zeros(2, 1, heads, maxlen, 80, dtype=torch.int8, device="cuda")
    x = torch.randn(1, 3, heads, 128, generator=torch.Generator().manual_seed(8))
    at = torch.tensor([maxlen - 3], dtype=torch.int32, device="cuda")
    llmops.cache_write_q4(x.cuda(), x.cuda(), cache, at, 0)
    want = ref.quantise(x[0].numpy()).transpose(1, 0, 2)
    for plane in (0, 1):
        _same(cache[plane, 0, :, -3:], want)
    got = llmops.cache_read_q4(cache, 4, starts=at - 1)[:, 0]
    assert np.array_equal(got[1, :, 1:].cpu().double().numpy(), ref.values(want)) and not got[:, :, 0].any()


def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(9)
    B, L, Hkv, maxlen = 2, 5, 4, 60
    k, v = torch.randn(B, L, Hkv * 128, generator=g).cuda(), torch.randn(B, L, Hkv * 128, generator=g).cuda()
    lengths, f = torch.zeros(B, dtype=torch.int32, device="cuda"), _inv_freq().cuda()
    cache = torch.zeros(2, B, Hkv, maxlen, 80, dtype=torch.int8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        llmops.cache_write_q4(k, v, cache, lengths, 0, inv_freq=f)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            llmops.cache_write_q4(k, v, cache, lengths, 0, inv_freq=f)
            got = llmops.cache_read_q4(cache, L, starts=lengths)
    torch.cuda.synchronize()
    for step in range(4):
        k.copy_(torch.randn(B, L, Hkv * 128, generator=g)), lengths.copy_(torch.tensor([7 * step, 55 - 3 * step]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.zeros_like(cache)
        llmops.cache_write_q4(k, v, want, lengths, 0, inv_freq=f)
        assert torch.equal(got, llmops.cache_read_q4(want, L, starts=lengths))


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    cache, lengths = z(2, 2, 4, 8, 80, dtype=torch.int8), z(2, dtype=torch.int32)
    k = z(2, 3, 512)
    ok = lambda **kw: llmops.cache_write_q4(**{**dict(k=k, v=k, kv_cache=cache, lengths=lengths, layer_id=0), **kw})  # noqa: E731
    ok()
    for kw in (dict(k=z(2, 3, 256)), dict(v=z(2, 2, 512)), dict(k=k.half()), dict(k=k.bfloat16(), v=k.bfloat16()), dict(kv_cache=z(2, 2, 4, 8, 80)), dict(kv_cache=cache[..., :64]),
               dict(kv_cache=cache[:, :1]), dict(kv_cache=cache.transpose(1, 2)), dict(lengths=lengths[:1]), dict(lengths=lengths.long()), dict(q_lens=lengths[:1]),
               dict(layer_id=1), dict(layer_id=-1), dict(inv_freq=z(65)), dict(inv_freq=z(64).double()), dict(k=z(2, 3, 1024)[..., ::2]), dict(k=z(2, 3, 513)[..., 1:]),
               dict(k=k.cpu()), dict(lengths=lengths.cpu())):
        with pytest.raises(RuntimeError):
            ok(**kw)
    with pytest.raises(RuntimeError):  # rows that lie in the cache
        ok(k=cache.view(torch.float32).flatten().as_strided((2, 3, 512), (512, 0, 1)), v=k)
    for kw in (dict(kv_cache=cache.float()), dict(rows=-1), dict(dtype=torch.bfloat16), dict(starts=lengths[:1]), dict(starts=lengths.long())):
        with pytest.raises(RuntimeError):
            llmops.cache_read_q4(**{**dict(kv_cache=cache, rows=3), **kw})


def test_frequencies_of_no_dims_are_refused():
    """no frequencies are None: an empty tensor of them does not stand for rows that come rotated"""
    cache, lengths, k = torch.full((2, 1, 4, 8, 80), 3, dtype=torch.int8, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.ones(1, 3, 512, device="cuda")
    native = llmops._lib.host()
    for host in (native, llmops._lib._PythonCalls()):
        llmops._lib._host = host
        try:
            with pytest.raises(RuntimeError, match="inv_freq"):
                llmops.cache_write_q4(k, k, cache, lengths, 0, inv_freq=torch.zeros(0, device="cuda"))
        finally:
            llmops._lib._host = native
    assert (cache == 3).all()


@pytest.mark.parametrize("offset,spread", [(0.0, 1.0), (1000.0, 0.5), (-60000.0, 100.0), (3.0, 1e-3), (1e-4, 1e-6), (2.0 ** -14, 2.0 ** -20), (0.0, 2.0 ** -22), (-7.0, 0.0)])
def test_how_far_a_value_may_be_off(offset, spread):
    """With u the group's unit: levels lie s <= range / (15 u) + 1 units apart, and the ends half a unit inside at most, so that a value is off by at most (range / 15 + u) / 2;
    u is at most a 1016th of the largest magnitude, or 2^-24.  A group whose values have much in common is off by the second part."""
    g = torch.Generator().manual_seed(13)
    x = offset + spread * torch.randn(300, 128, generator=g)
    back = llmops.cache_read_q4(_write_one(x), 300, dtype=torch.float32)[0, 0, 0].cpu().double().reshape(300, 4, 32)
    t = x.double().reshape(300, 4, 32)
    span, most = t.amax(-1) - t.amin(-1), t.abs().amax(-1)
    off = (back - t).abs().amax(-1)
    assert (off <= span / 30 + torch.clamp(most / 2032, min=2.0 ** -25)).all()
    if offset == 1000.0:  # (a thirtieth of the range alone is no bound)
        assert float((off / span).max()) > 0.1
