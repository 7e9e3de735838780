"""No-GPU checks of the entry points for several requests: bad arguments are refused before anything touches the device, workspaces
are sized by host arithmetic, and the Python functions refuse host tensors."""
import ctypes

import pytest
import torch

import llmops
from llmops import _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


P = ctypes.c_void_p(4096)  # (an aligned address that is never followed: there is no device here, a launch would be a HIP error)
NONE = ctypes.c_void_p(0)


def _refused(lib, rc, what, code=1):
    assert rc == code and what in lib.llmops_last_error(), (rc, lib.llmops_last_error())


def _prefix(lib, **kw):
    a = dict(q=P, qb=4096, ql=4096, k=P, kb=4096, kl=4096, v=P, vb=4096, vl=4096, B=2, qL=3, H=32, Hkv=8, S=128, f=P, half=64, pc=P, pplanes=2, pmax=100, plen=50,
             kv=ctypes.c_void_p(1 << 40), dt=0, planes=2, maxlen=64, lengths=P, q_lens=NONE, layer=0, out=P, ws=P, bytes=1 << 40, stream=NONE)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.llmops_attention_rope_prefix(*a.values())


@pytest.mark.parametrize("kw,what", [
    (dict(q=NONE), b"q != nullptr"), (dict(out=NONE), b"out != nullptr"), (dict(lengths=NONE), b"lengths != nullptr"), (dict(pc=NONE), b"prefix_cache != nullptr"),
    (dict(S=64), b"S == 128"), (dict(H=30), b"prefix_sizes_fit"), (dict(Hkv=0), b"prefix_sizes_fit"), (dict(B=0), b"prefix_sizes_fit"), (dict(qL=0), b"prefix_sizes_fit"),
    (dict(B=1 << 20, qL=1 << 10), b"prefix_sizes_fit"), (dict(plen=1 << 24, pmax=1 << 24), b"prefix_sizes_fit"), (dict(plen=-1), b"prefix_sizes_fit"),
    (dict(plen=101), b"prefix_len <= prefix_maxlen"), (dict(half=65), b"2 * half <= S"), (dict(half=0), b"half > 0"), (dict(layer=1), b"layer_id"), (dict(layer=-1), b"layer_id"),
    (dict(B=1 << 22, qL=2, H=16, Hkv=1, maxlen=1, kv=ctypes.c_void_p(1 << 56)), b"merge < most"), (dict(B=(1 << 24) - 1, qL=2, H=1, Hkv=1, maxlen=1, pc=NONE, plen=0), b"prep < most"),
    (dict(layer=1, planes=4), b"prefix_planes"), (dict(dt=2), b"cache_dtype"), (dict(q=ctypes.c_void_p(4104)), b"aligned(q, 16)"), (dict(ws=ctypes.c_void_p(4112)), b"aligned(workspace, 256)"),
    (dict(kl=1026), b"k_stride_l % 4 == 0"), (dict(kv=P), b"p1 <= o0"), (dict(kv=ctypes.c_void_p(4096 + 4 * 1024 * 8)), b"p1 <= o0"),
])
def test_attention_rope_prefix_refuses(lib, kw, what):
    _refused(lib, _prefix(lib, **kw), what)


def test_attention_rope_prefix_workspace(lib):
    need = lib.llmops_attention_prefix_workspace_bytes(2, 3, 32, 8, 128, 50, 64)
    assert need > 2 * 3 * 32 * 128 * 4  # at least the rotated queries
    _refused(lib, _prefix(lib, bytes=need - 1), b"workspace bytes", 2)
    _refused(lib, _prefix(lib, ws=NONE), b"workspace != nullptr")
    assert lib.llmops_attention_prefix_workspace_bytes(2, 3, 32, 8, 64, 50, 64) == 0
    assert lib.llmops_attention_prefix_workspace_bytes(2, 3, 32, 5, 128, 50, 64) == 0


def _lora(lib, **kw):
    a = dict(y=P, yb=100, yl=100, x=P, xb=100, xl=100, B=4, M=2, N=64, K=96, A=P, W=P, dt=1, R=16, n=3, ids=P, scales=P, out=P, ob=100, ol=100, ws=P, bytes=1 << 40,
             stream=NONE)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.llmops_lora_add(*a.values())


@pytest.mark.parametrize("kw,what", [
    (dict(y=NONE), b"y != nullptr"), (dict(ids=NONE), b"ids != nullptr"), (dict(out=NONE), b"out != nullptr"), (dict(B=0), b"lora_sizes_fit"), (dict(M=-1), b"lora_sizes_fit"),
    (dict(N=0), b"lora_sizes_fit"), (dict(K=0), b"lora_sizes_fit"), (dict(R=0), b"lora_sizes_fit"), (dict(R=4097), b"lora_sizes_fit"), (dict(B=1 << 12, M=1 << 9), b"lora_sizes_fit"),
    (dict(n=0), b"adapters > 0"), (dict(dt=3), b"weight_dtype"), (dict(A=ctypes.c_void_p(4097)), b"aligned(lora_A, e)"), (dict(x=ctypes.c_void_p(4098)), b"aligned(x, 4)"),
    (dict(W=ctypes.c_void_p(4098), dt=0), b"aligned(lora_B, e)"), (dict(N=1 << 29), b"lora_sizes_fit"), (dict(K=1 << 29), b"lora_sizes_fit"),
])
def test_lora_add_refuses(lib, kw, what):
    _refused(lib, _lora(lib, **kw), what)


def test_lora_add_workspace(lib):
    for B, M, K, R, n in ((4, 2, 96, 16, 3), (1, 1, 4096, 8, 1), (1, 2048, 11008, 64, 1), (64, 1, 4096, 100, 64), (300, 20, 5000, 7, 9)):
        need = lib.llmops_lora_workspace_bytes(B, M, 64, K, R, n)
        row = (R + 3) // 4 * 16
        assert need >= B * M * row and need % (B * M * row) == 0  # (whole runs of K, a row of sums in whole fours)
        _refused(lib, _lora(lib, B=B, M=M, K=K, R=R, n=n, bytes=need - 1), b"workspace bytes", 2)
    _refused(lib, _lora(lib, ws=NONE), b"workspace bytes", 2)
    assert lib.llmops_lora_workspace_bytes(0, 1, 1, 1, 1, 1) == 0 and lib.llmops_lora_workspace_bytes(1, 1, 1, 1, 1, 0) == 0


def _verify(lib, **kw):
    a = dict(z=P, B=2, K=3, V=100, d=P, q=P, u=P, t=NONE, one=ctypes.c_float(1.0), n=NONE, tokens=P, accepted=P, ws=P, bytes=1 << 40, stream=NONE)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.llmops_verify_drafts(*a.values())


@pytest.mark.parametrize("kw,what", [
    (dict(z=NONE), b"logits != nullptr"), (dict(u=NONE), b"uniforms != nullptr"), (dict(tokens=NONE), b"tokens != nullptr"), (dict(d=NONE), b"drafts != nullptr"),
    (dict(B=0), b"verify_sizes_fit"), (dict(K=-1), b"verify_sizes_fit"), (dict(V=0), b"verify_sizes_fit"), (dict(V=(1 << 27) + 1), b"verify_sizes_fit"),
    (dict(B=1 << 20, K=15), b"verify_sizes_fit"), (dict(B=1 << 20, V=1 << 16), b"a.runs < "), (dict(d=ctypes.c_void_p(4100)), b"aligned(drafts, 8)"), (dict(ws=ctypes.c_void_p(4104)), b"aligned(workspace, 16)"),
])
def test_verify_drafts_refuses(lib, kw, what):
    _refused(lib, _verify(lib, **kw), what)


def test_verify_drafts_workspace(lib):
    need = lib.llmops_verify_drafts_workspace_bytes(2, 3, 100)
    assert need > 0
    _refused(lib, _verify(lib, bytes=need - 1), b"workspace bytes", 2)
    _refused(lib, _verify(lib, ws=NONE), b"workspace bytes", 2)
    assert lib.llmops_verify_drafts_workspace_bytes(2, 3, 0) == 0


def test_host_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(RuntimeError, match="HIP device"):
        llmops.attention_rope_prefix(z(1, 1, 128), z(1, 1, 128), z(1, 1, 128), z(64), None, 0, z(2, 1, 1, 4, 128), z(1, dtype=torch.int32), 0)
    with pytest.raises(RuntimeError, match="HIP device"):
        llmops.lora_add(z(1, 1, 8), z(1, 1, 8), z(1, 8, 8), z(1, 8, 8), z(1, dtype=torch.int32), z(1))
    with pytest.raises(RuntimeError, match="HIP device"):
        llmops.verify_drafts(z(1, 1, 8), z(1, 0, dtype=torch.int64), z(1, 1))


def test_request_cache_bookkeeping_on_the_host():
    from llmops.opset import PrefixCache
    cfg = dict(layer_num=1, head_num=2, head_size=128)
    c = PrefixCache(cfg, 3, 10, device="cpu")
    c.keep(4)
    c.keep(torch.tensor([1, 7, 0], dtype=torch.int32))
    assert c.lengths.tolist() == [5, 10, 4] and c.size() == c.cache.numel() * 4 and c.prefix_len == 0
    c.forget(1)
    c.forget(0, 2)
    assert c.lengths.tolist() == [2, 0, 4]
    with pytest.raises(ValueError):
        c.forget(0, 11)


@pytest.mark.parametrize("prefix,maxlen", [(0, 1 << 24), (1 << 23, 1 << 23), ((1 << 24) - 1, 1)])
def test_attention_rope_prefix_up_to_the_last_position(lib, prefix, maxlen):
    """prefix and own rows together up to 2^24, as documented: the sizes are taken (refused is the workspace), and one row more is not"""
    need = lib.llmops_attention_prefix_workspace_bytes(2, 3, 32, 8, 128, prefix, maxlen)
    assert need > 0 and lib.llmops_attention_prefix_workspace_bytes(2, 3, 32, 8, 128, prefix, maxlen + 1) == 0
    kw = dict(plen=prefix, pmax=1 << 24, maxlen=maxlen, kv=ctypes.c_void_p(1 << 50), bytes=need - 1)
    _refused(lib, _prefix(lib, **kw), b"workspace bytes", 2)
    kw["maxlen"] += 1
    _refused(lib, _prefix(lib, **kw), b"prefix_sizes_fit")


@pytest.mark.parametrize("kw,what", [
    # (y, x and out: 4 sequences of 2 tokens, 100 fp32 values apart each way unless said; y and out 64 wide, x 96)
    (dict(), b"rows_apart(out_rows)"), (dict(ob=200, ol=63), b"rows_apart(out_rows)"), (dict(ob=0, ol=64), b"rows_apart(out_rows)"), (dict(ob=64, ol=64), b"rows_apart(out_rows)"),
    (dict(ob=200), b"apart(out_rows, x_rows)"), (dict(ob=200, yb=200), b"apart(out_rows, x_rows)"),
    (dict(ob=400, ol=200, yb=400, yl=200, xb=400, xl=200, x=ctypes.c_void_p(4096 + 4 * 63)), b"apart(out_rows, x_rows)"),
    (dict(ob=400, ol=200, yb=400, yl=200, xb=400, xl=200, x=ctypes.c_void_p(4096 + 4 * 110)), b"apart(out_rows, x_rows)"),
    (dict(ob=400, ol=200, yb=400, yl=200, xb=0, xl=0, x=ctypes.c_void_p(4096 + 4 * 1390)), b"apart(out_rows, x_rows)"),
    (dict(ob=200, yb=201, x=ctypes.c_void_p(1 << 20)), b"in_place || apart(out_rows, y_rows)"),
    (dict(ob=200, yb=200, x=ctypes.c_void_p(1 << 20), y=ctypes.c_void_p(4100)), b"in_place || apart(out_rows, y_rows)"),
    (dict(ob=200, yb=200, x=ctypes.c_void_p(1 << 20), y=ctypes.c_void_p(4096 + 4 * 363)), b"in_place || apart(out_rows, y_rows)"),
    (dict(B=1, M=1, x=ctypes.c_void_p(1 << 20), y=ctypes.c_void_p(4096 - 4 * 63)), b"in_place || apart(out_rows, y_rows)"),
])
def test_lora_add_refuses_an_output_over_its_inputs(lib, kw, what):
    _refused(lib, _lora(lib, **kw), what)


@pytest.mark.parametrize("kw,what", [
    # q [2, 3, 32 heads] and out dense, k and v [2, 3, 8 heads], cache [2, 2, 8, 64, 128]: 2 * 8 * 64 * 128 = 2^17 values a plane, 2^18 a layer
    (dict(kv=ctypes.c_void_p((1 << 30) - 4 * (1 << 18) + 16)), b"apart(own, q)"), (dict(k=ctypes.c_void_p((1 << 40) + 4 * ((1 << 18) - 4))), b"apart(own, k)"),
    (dict(v=ctypes.c_void_p((1 << 40) - 4 * (5 * 1024 + 1024 - 4)), vb=3072, vl=1024), b"apart(own, v)"), (dict(layer=1, planes=4, pplanes=4, v=ctypes.c_void_p((1 << 40) + 4 * (1 << 18))), b"apart(own, v)"),
    (dict(out=ctypes.c_void_p(1 << 30)), b"apart(out, q)"), (dict(out=ctypes.c_void_p((1 << 30) + 4 * 4092), qb=12288), b"apart(out, q)"),
    (dict(out=ctypes.c_void_p((1 << 31) + 4 * 1020)), b"apart(out, k)"), (dict(out=ctypes.c_void_p((1 << 32) - 16)), b"apart(out, v)"),
    (dict(out=ctypes.c_void_p(1 << 40)), b"apart(out, own)"), (dict(out=ctypes.c_void_p(4096)), b"apart(out, prefix)"),
])
def test_attention_rope_prefix_refuses_outputs_over_inputs(lib, kw, what):
    a = dict(q=ctypes.c_void_p(1 << 30), k=ctypes.c_void_p(1 << 31), v=ctypes.c_void_p(1 << 32), out=ctypes.c_void_p(1 << 33))
    a.update(kw)
    _refused(lib, _prefix(lib, **a), what)


@pytest.mark.parametrize("kw,what", [
    # 2 sequences, 3 drafts, 100 tokens: logits [2, 4, 100], probabilities [2, 3, 100], tokens [2, 4] int64
    (dict(d=1 << 20), b"apart(out, drafts_at)"), (dict(d=(1 << 20) - 40), b"apart(out, drafts_at)"), (dict(z=(1 << 20) - 3196), b"apart(out, logits_at)"), (dict(u=(1 << 20) + 60), b"apart(out, random_at)"),
    (dict(q=(1 << 20) - 2396), b"apart(out, probs_at)"), (dict(t=(1 << 21) + 4), b"apart(out, temperatures_at)"), (dict(n=1 << 21), b"apart(out, lens_at)"), (dict(accepted=(1 << 20) + 60), b"apart(first, second)"),
])
def test_verify_drafts_refuses_outputs_over_inputs(lib, kw, what):
    at = dict(z=1 << 30, d=1 << 31, q=1 << 32, u=1 << 33, t=1 << 34, n=1 << 35, tokens=1 << 20, accepted=1 << 21)
    at.update(kw)
    _refused(lib, _verify(lib, **{name: ctypes.c_void_p(x) for name, x in at.items()}), what)
