"""No-GPU checks of the entry points for a cache in 4 bits and for log probabilities: bad arguments are refused before anything touches the
device, workspaces are sized by host arithmetic, and the Python functions refuse host tensors."""
import ctypes

import pytest
import torch

import llmops
from llmops import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = ctypes.c_void_p(4096)  # (an aligned address that is never followed: there is no device here, a launch would be a HIP error)
FAR = ctypes.c_void_p(1 << 40)
NONE = ctypes.c_void_p(0)


def _refused(lib, rc, what, code=1):
    assert rc == code and what in lib.llmops_last_error(), (rc, lib.llmops_last_error())


def _call(fn, defaults, kw):
    assert set(kw) <= set(defaults)
    return fn(*{**defaults, **kw}.values())


def _write(lib, **kw):
    return _call(lib.llmops_cache_write_q4, dict(k=P, kb=1024, kl=1024, kh=128, v=P, vb=1024, vl=1024, vh=128, dt=0, B=2, qL=3, Hkv=8, S=128, f=P, half=64, kv=FAR, planes=2,
                                                 maxlen=64, lengths=P, q_lens=NONE, layer=0, stream=NONE), kw)


@pytest.mark.parametrize("kw,what", [
    (dict(k=NONE), b"k != nullptr"), (dict(kv=NONE), b"kv_cache != nullptr"), (dict(lengths=NONE), b"lengths != nullptr"), (dict(S=64), b"S == 128"), (dict(dt=2), b"dtype"),
    (dict(B=0), b"B > 0"), (dict(qL=0), b"qL > 0"), (dict(Hkv=0), b"Hkv > 0"), (dict(maxlen=0), b"maxlen > 0"), (dict(maxlen=(1 << 24) + 1), b"maxlen"), (dict(half=65), b"half"),
    (dict(half=0), b"half"), (dict(layer=1), b"layer_id"), (dict(layer=-1), b"layer_id"), (dict(k=ctypes.c_void_p(4104)), b"aligned(k, 16)"),
    (dict(kv=ctypes.c_void_p(4104)), b"aligned"), (dict(kl=1026), b"k_stride_l"), (dict(dt=1, vh=132), b"v_stride_h"), (dict(kv=P), b"apart(written, kh)"),
    (dict(k=ctypes.c_void_p(1 << 30), kv=ctypes.c_void_p((1 << 30) - 2 * 2 * 8 * 64 * 80 + 16)), b"apart(written"), (dict(B=1 << 20, qL=1 << 20, maxlen=1), b"most"),
    (dict(lengths=ctypes.c_void_p((1 << 40) + 400)), b"apart(written, lengths_at)"), (dict(q_lens=FAR), b"apart(written, q_lens_at)"), (dict(f=FAR), b"apart(written, inv_freq_at)"),
])
def test_cache_write_refuses(lib, kw, what):
    _refused(lib, _write(lib, **kw), what)


def test_cache_write_between_what_it_reads(lib):
    # rows of the cache between k's heads, which lie apart: not refused for that (there is no device: the launch fails)
    rc = _write(lib, kh=1 << 20, kb=0, kl=128, v=ctypes.c_void_p(1 << 41), kv=ctypes.c_void_p(4096 + (1 << 19)), B=1, maxlen=8)
    assert rc == 3 or (rc == 0 and torch.cuda.is_available())


def _read(lib, **kw):
    return _call(lib.llmops_cache_read_q4, dict(kv=FAR, planes=2, B=2, Hkv=8, maxlen=64, S=128, starts=NONE, rows=10, out=P, dt=1, stream=NONE), kw)


@pytest.mark.parametrize("kw,what", [
    (dict(kv=NONE), b"kv_cache != nullptr"), (dict(out=NONE), b"out != nullptr"), (dict(S=64), b"S == 128"), (dict(dt=2), b"dtype"), (dict(rows=0), b"rows > 0"), (dict(planes=0), b"planes > 0"),
    (dict(out=ctypes.c_void_p(4104)), b"aligned"), (dict(out=FAR), b"apart(out_at, cache_at)"), (dict(starts=P), b"apart(out_at, starts_at)"), (dict(rows=1 << 24, B=64), b"most"),
])
def test_cache_read_refuses(lib, kw, what):
    _refused(lib, _read(lib, **kw), what)


def _attend(lib, **kw):
    return _call(lib.llmops_attention_rope_q4, dict(q=P, qb=4096, ql=4096, k=P, kb=4096, kl=4096, v=P, vb=4096, vl=4096, B=2, qL=3, H=32, Hkv=8, S=128, f=P, half=64, kv=FAR,
                                                    planes=2, maxlen=640, lengths=P, q_lens=NONE, layer=0, out=ctypes.c_void_p(1 << 30), ws=ctypes.c_void_p(1 << 35),
                                                    bytes=1 << 40, stream=NONE), kw)


@pytest.mark.parametrize("kw,what", [
    (dict(q=NONE), b"q != nullptr"), (dict(out=NONE), b"out != nullptr"), (dict(ws=NONE), b"workspace != nullptr"), (dict(lengths=NONE), b"lengths != nullptr"), (dict(S=64), b"S == 128"),
    (dict(H=30), b"q4_sizes_fit"), (dict(Hkv=0), b"q4_sizes_fit"), (dict(B=0), b"q4_sizes_fit"), (dict(qL=0), b"q4_sizes_fit"), (dict(maxlen=0), b"q4_sizes_fit"),
    (dict(maxlen=(1 << 24) + 1), b"q4_sizes_fit"), (dict(B=1 << 20), b"q4_sizes_fit"), (dict(B=1 << 12, maxlen=1 << 24), b"q4_sizes_fit"), (dict(half=65), b"half"), (dict(half=0), b"half"),
    (dict(layer=1), b"layer_id"), (dict(layer=-1), b"layer_id"), (dict(q=ctypes.c_void_p(4104)), b"aligned(q, 16)"), (dict(ws=ctypes.c_void_p((1 << 35) + 16)), b"aligned(workspace, 256)"),
    (dict(kl=1026), b"k_stride_l"), (dict(kv=P), b"apart(written, q_at)"), (dict(out=P), b"apart(out_at, q_at)"), (dict(out=FAR), b"apart(out_at, written)"),
    (dict(lengths=FAR), b"apart(written, lengths_at)"), (dict(q_lens=FAR), b"apart(written, q_lens_at)"), (dict(f=FAR), b"apart(written, inv_freq_at)"),
    (dict(lengths=ctypes.c_void_p(1 << 30)), b"apart(out_at, lengths_at)"), (dict(q_lens=ctypes.c_void_p(1 << 30)), b"apart(out_at, q_lens_at)"),
    (dict(f=ctypes.c_void_p((1 << 30) + 256)), b"apart(out_at, inv_freq_at)"),
])
def test_attention_refuses(lib, kw, what):
    _refused(lib, _attend(lib, **kw), what)


def test_attention_workspace(lib):
    for B, qL, H, Hkv, maxlen in ((2, 3, 32, 8, 640), (1, 1, 1, 1, 1), (64, 1, 32, 32, 100000), (4, 300, 32, 32, 1777), (1, 17, 8, 8, 384), (300, 2, 4, 1, 5000)):
        need = lib.llmops_attention_q4_workspace_bytes(B, qL, H, Hkv, 128, maxlen)
        assert need > 0
        kw = dict(B=B, qL=qL, H=H, Hkv=Hkv, maxlen=maxlen, out=ctypes.c_void_p(1 << 45), kv=ctypes.c_void_p(1 << 46))
        _refused(lib, _attend(lib, bytes=need - 1, **kw), b"workspace bytes", 2)
    assert lib.llmops_attention_q4_workspace_bytes(2, 3, 32, 8, 64, 640) == 0 and lib.llmops_attention_q4_workspace_bytes(2, 3, 32, 5, 128, 640) == 0


def _logprobs(lib, **kw):
    return _call(lib.llmops_token_logprobs, dict(z=FAR, sb=300, sl=100, B=2, L=3, V=100, t=P, tb=3, tl=1, top=5, lp=ctypes.c_void_p(8192), ent=ctypes.c_void_p(12288),
                                                 ids=ctypes.c_void_p(16384), lps=ctypes.c_void_p(20480), ws=ctypes.c_void_p(1 << 35), bytes=1 << 40, stream=NONE), kw)


@pytest.mark.parametrize("kw,what", [
    (dict(z=NONE), b"logits != nullptr"), (dict(t=NONE), b"tokens != nullptr"), (dict(lp=NONE), b"logprobs != nullptr"), (dict(ent=NONE), b"entropy != nullptr"),
    (dict(ids=NONE), b"top_tokens != nullptr"), (dict(lps=NONE), b"top_logprobs != nullptr"), (dict(B=0), b"logprob_sizes_fit"), (dict(L=0), b"logprob_sizes_fit"),
    (dict(V=0), b"logprob_sizes_fit"), (dict(V=(1 << 27) + 1), b"logprob_sizes_fit"), (dict(top=65), b"logprob_sizes_fit"), (dict(top=-1), b"logprob_sizes_fit"),
    (dict(V=4), b"logprob_sizes_fit"), (dict(B=1 << 13, L=1 << 11), b"logprob_sizes_fit"), (dict(B=1 << 12, L=1 << 11, V=1 << 16), b"w.runs"), (dict(t=ctypes.c_void_p(4100)), b"aligned"),
    (dict(z=ctypes.c_void_p(4098)), b"aligned"), (dict(lp=ctypes.c_void_p(12288)), b"apart"), (dict(ent=P), b"apart(out[i], tokens_at)"), (dict(ids=FAR), b"apart(out[i], logits_at)"),
    (dict(lps=ctypes.c_void_p(16384)), b"apart"), (dict(ws=ctypes.c_void_p((1 << 35) + 8)), b"aligned(workspace, 16)"),
])
def test_token_logprobs_refuses(lib, kw, what):
    _refused(lib, _logprobs(lib, **kw), what)


def test_token_logprobs_workspace(lib):
    for B, L, V, top in ((2, 3, 100, 5), (1, 1, 55296, 64), (3, 700, 32003, 0), (1, 1, 1, 1)):
        need = lib.llmops_token_logprobs_workspace_bytes(B, L, V, top)
        assert need >= B * L * 16
        kw = dict(B=B, L=L, V=V, top=top, lp=ctypes.c_void_p(1 << 41), ent=ctypes.c_void_p(1 << 42), ids=ctypes.c_void_p(1 << 43), lps=ctypes.c_void_p(1 << 44))
        _refused(lib, _logprobs(lib, bytes=need - 1, **kw), b"workspace bytes", 2)
        _refused(lib, _logprobs(lib, ws=NONE, **kw), b"workspace bytes", 2)
    assert lib.llmops_token_logprobs_workspace_bytes(0, 1, 1, 0) == 0 and lib.llmops_token_logprobs_workspace_bytes(1, 1, 3, 4) == 0


def test_python_functions_refuse_host_tensors():
    cache, lengths, k = torch.zeros(2, 1, 2, 8, 80, dtype=torch.int8), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 256)
    for call in (lambda: llmops.cache_write_q4(k, k, cache, lengths, 0), lambda: llmops.cache_read_q4(cache, 3),
                 lambda: llmops.attention_rope_q4(k, k, k, torch.ones(64), cache, lengths, 0), lambda: llmops.token_logprobs(torch.zeros(1, 1, 5), torch.zeros(1, 1, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="no CPU path|HIP device"):
            call()


@pytest.mark.parametrize("B,qL,H,Hkv,maxlen,fits", [
    (1, 100000, 32, 32, 100000, True), (1, 100000, 32, 8, 1 << 20, True),                       # long prompts: tiles of 64 queries count
    (1, 4096, 32, 32, 16383 * 128, True), (1, 4096, 32, 1, 1 << 21, True),
    (1 << 14, 1, 1, 1, 131070 * 128, True), (1 << 14, 1, 1, 1, 131070 * 128 + 1, False),        # 2^31 units less 2^14, and 2^31
    (1 << 12, 64, 4, 4, 131070 * 128, True), (1 << 12, 65, 4, 4, 65535 * 128, False), (1 << 12, 65, 4, 4, 65534 * 128, True),
    (1 << 23, 1, 1, 1, 254 * 128, True), (1 << 23, 1, 1, 1, 255 * 128, False), (1, 1 << 19, 32, 32, 1, False), (1, (1 << 19) - 1, 32, 32, 1, True)])
def test_attention_sizes_that_fit(lib, B, qL, H, Hkv, maxlen, fits):
    need = lib.llmops_attention_q4_workspace_bytes(B, qL, H, Hkv, 128, maxlen)
    assert (need > 0) == fits
    far = dict(B=B, qL=qL, H=H, Hkv=Hkv, maxlen=maxlen, out=ctypes.c_void_p(1 << 55), kv=ctypes.c_void_p(1 << 56), qb=0, ql=0, kb=0, kl=0, vb=0, vl=0)
    _refused(lib, _attend(lib, bytes=0, **far), *((b"workspace bytes", 2) if fits else (b"q4_sizes_fit",)))
