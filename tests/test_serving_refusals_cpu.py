"""Refusals of the serving and distillation entry points: wrong sizes, types and pointers never reach a launch (no GPU needed)."""
import pytest
import torch

from neko_amd import _lib, ops

E4, I8, BF16 = torch.float8_e4m3fn, torch.int8, torch.bfloat16
P = 0x10000            # a non-null, aligned address that no refused call looks at


def _rc(name, args):
    return getattr(_lib.load(), name)(*args)


APPEND = dict(k8=P, v8=P, ks=P, vs=P, dtype=0, S=2, H=2, cap=64, hd=32, block=16, k=P, k_ss=64, k_st=64, v=P, v_ss=64, v_st=64, pos=P, n_new=None, T=1, stream=None)
READ = dict(k8=P, v8=P, ks=P, vs=P, dtype=0, S=2, H=2, cap=64, hd=32, block=16, length=P, L=64, k=P, v=P, stream=None)
ATTN = dict(k8=P, v8=P, ks=P, vs=P, dtype=0, S=2, H=2, cap=64, hd=32, block=16, q=P, q_ss=64, q_st=64, out=P, o_ss=64, o_st=64, G=1, T=1, pos=P, n_new=None,
            start=None, window=0, sinks=0, scale=1.0, max_len=0, ws=None, ws_floats=0, stream=None)
VERIFY = dict(target=P, t_sb=10, t_sr=10, draft=None, d_sb=0, d_sr=0, is_bf16=0, B=1, K=2, V=10, tokens=P, u=P, r=P, n_draft=None, temperature=1.0, acc=P, out=P,
              ws=P, ws_bytes=1 << 20, stream=None)
DISTILL = dict(z=P, ldz=16, is_bf16=1, R=1, V=10, Vpad=16, t_val=P, t_idx=P, k=4, weight=P, tau=1.0, target=P, hard=0.5, loss=P, dl=P, ldd=16, stream=None)

BAD_CACHE = [dict(k8=None), dict(v8=None), dict(ks=None), dict(vs=None), dict(dtype=2), dict(dtype=-1), dict(S=0), dict(H=0), dict(cap=0), dict(cap=65),
             dict(cap=1 << 25), dict(hd=48), dict(hd=256), dict(block=8), dict(block=128), dict(S=70000), dict(H=70000)]


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(k=None), dict(v=None), dict(pos=None), dict(T=0), dict(k=P + 8), dict(v_st=60), dict(k_ss=4)], ids=str)
def test_append_refuses(bad):
    assert _rc("neko_kv8_append", {**APPEND, **bad}.values()) in (-1, -2)


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(length=None), dict(k=None), dict(v=None), dict(L=0), dict(L=65)], ids=str)
def test_read_refuses(bad):
    assert _rc("neko_kv8_read", {**READ, **bad}.values()) in (-1, -2)


@pytest.mark.parametrize("bad", BAD_CACHE + [dict(q=None), dict(out=None), dict(pos=None), dict(G=0), dict(T=0), dict(T=65), dict(window=-1), dict(sinks=-1),
                                             dict(q=P + 2), dict(o_st=63), dict(scale=0.0), dict(scale=float("nan")), dict(cap=1 << 16, S=1), dict(G=1 << 24, T=2)], ids=str)
def test_attn_refuses(bad):
    """(the long cache without a workspace among them: its key axis is split)"""
    assert _rc("neko_attn_kv8", {**ATTN, **bad}.values()) in (-1, -2)


@pytest.mark.parametrize("bad", [dict(target=None), dict(tokens=None), dict(acc=None), dict(out=None), dict(ws=None), dict(B=0), dict(K=0), dict(V=0), dict(K=63),
                                 dict(B=70000), dict(u=None), dict(r=None), dict(temperature=-1.0), dict(temperature=float("nan")), dict(ws_bytes=8), dict(ws=P + 4)], ids=str)
def test_verify_refuses(bad):
    assert _rc("neko_verify_draft", {**VERIFY, **bad}.values()) in (-1, -2)


@pytest.mark.parametrize("bad", [dict(z=None), dict(weight=None), dict(R=0), dict(V=0), dict(Vpad=9), dict(Vpad=12), dict(ldz=8), dict(ldz=18), dict(z=P + 2), dict(ldd=8),
                                 dict(dl=P + 4), dict(tau=0.0), dict(tau=float("nan")), dict(hard=-0.1), dict(hard=1.1), dict(target=None), dict(t_val=None),
                                 dict(t_idx=None), dict(k=0), dict(k=1025), dict(loss=None, dl=None)], ids=str)
def test_distill_refuses(bad):
    assert _rc("neko_distill_topk", {**DISTILL, **bad}.values()) in (-1, -2)


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.neko_attn_kv8_ws_floats(0, 1, 1, 64, 32, 1, 0, 0, 0) == 0 and lib.neko_attn_kv8_ws_floats(64, 24, 1, 64, 32, 1, 0, 0, 0) == 0
    assert lib.neko_attn_kv8_ws_floats(1, 1, 1, 8192, 128, 1, 0, 0, 0) > 0 and lib.neko_attn_kv8_ws_floats(1, 1, 1, 8192, 128, 1, 0, 0, 64) == 0
    assert lib.neko_attn_kv8_ws_floats(1, 1, 1, 8192, 128, 1, 50, 4, 0) == 0
    assert lib.neko_verify_draft_ws_bytes(0, 1, 1) == 0 and lib.neko_verify_draft_ws_bytes(2, 3, 5000) > 0


def _cache(dtype=E4, **k):
    return ops.KV8Cache(2, 3, 128, 64, dtype=dtype, device="cpu", **k)


def test_cache_shapes():
    c = _cache(I8, block=64)
    assert c.k.shape == (2, 3, 128, 64) and c.v.shape == (2, 3, 8, 64, 16) and c.k_scale.shape == (2, 3, 2) and c.v.dtype == I8
    d = ops.KV8Cache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
    assert (d.nseq, d.heads, d.cap, d.hd, d.block, d.dtype) == (2, 3, 128, 64, 64, I8) and d.k is c.k


@pytest.mark.parametrize("kw", [dict(cap=100), dict(cap=0), dict(hd=80), dict(block=48), dict(dtype=torch.uint8), dict(nseq=0)], ids=str)
def test_cache_refuses(kw):
    with pytest.raises(AssertionError):
        ops.KV8Cache(**{**dict(nseq=1, heads=1, cap=64, hd=32, device="cpu"), **kw})


def test_from_tensors_refuses():
    c = _cache()
    t = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale)
    for bad in (dict(v=c.v[:, :, :4]), dict(v=c.v.view(I8)), dict(k=c.k.transpose(2, 3)), dict(k_scale=c.k_scale.double()), dict(v_scale=c.v_scale[:, :, :2]),
                dict(k=c.k[:, :, :100]), dict(k=c.k.view(torch.uint8), v=c.v.view(torch.uint8)), dict(k_scale=c.k_scale[:, :, :1], v_scale=c.v_scale[:, :, :1])):
        with pytest.raises(AssertionError):
            ops.KV8Cache.from_tensors(**{**t, **bad})


def test_host_tensors_are_refused():
    """Every entry point insists on device tensors: there is no fallback."""
    c = _cache()
    x, pos = torch.zeros(2, 1, 3, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    z = torch.zeros(1, 16)
    for call in (lambda: ops.kv8_append(c, x, x, pos), lambda: ops.kv8_read(c, pos, 1), lambda: ops.attn_kv8(c, x, pos),
                 lambda: ops.verify_draft(torch.zeros(1, 2, 9), torch.zeros(1, 1, dtype=torch.int64), temperature=0.0),
                 lambda: ops.distill_topk(z, 9, 16, z[:, :4], torch.zeros(1, 4, dtype=torch.int32), torch.ones(1), dlogits=z)):
        with pytest.raises(AssertionError, match="device tensor"):
            call()


def test_plain_argument_errors():
    c = _cache()
    x, pos = torch.zeros(2, 1, 3, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.kv8_read(c, pos, 0), lambda: ops.kv8_read(c, pos, 129), lambda: ops.attn_kv8(c, x[:, :, :2], pos),
                 lambda: ops.verify_draft(torch.zeros(1, 2, 9), torch.zeros(1, 63, dtype=torch.int64)),
                 lambda: ops.verify_draft(torch.zeros(1, 2, 9), torch.zeros(1, 1, dtype=torch.int64), temperature=-1.0)):
        with pytest.raises(AssertionError):
            call()


@pytest.mark.parametrize("bad", [dict(q=P, out=P + 64, o_ss=64), dict(q=P, out=P + 64 * 1024, o_ss=32), dict(out=P + 64 * 1024, o_ss=0), dict(out=P + 128, o_ss=64),
                                 dict(T=2, q_ss=128, o_ss=128, out=P + 16), dict(T=2, q_ss=128, o_ss=64, o_st=64, out=P + (1 << 20)), dict(q_ss=-64), dict(o_ss=-64),
                                 dict(T=2, q_ss=256, q_st=128, o_ss=256, o_st=128, out=P + 64)], ids=str)
def test_attn_refuses_shared_rows(bad):
    """Output rows over one another or over rows of q that others still read."""
    assert _rc("neko_attn_kv8", {**ATTN, "out": P + (1 << 20), **bad}.values()) == -1


@pytest.mark.parametrize("bad", [dict(dl=P + 32), dict(dl=P + 16), dict(ldz=32, ldd=32, dl=P + 16), dict(ldz=32, ldd=32, dl=P + 48), dict(ldz=32), dict(tau=1e-39)], ids=str)
def test_distill_refuses_shared_rows(bad):
    assert _rc("neko_distill_topk", {**DISTILL, "R": 4, **bad}.values()) == -1


def test_verify_refuses_an_infinite_temperature():
    assert _rc("neko_verify_draft", {**VERIFY, "temperature": float("inf")}.values()) == -1


def test_verify_refuses_long_rows():
    assert _rc("neko_verify_draft", {**VERIFY, "V": (1 << 30) + 1, "ws_bytes": 1 << 40}.values()) == -2
    assert _lib.load().neko_verify_draft_ws_bytes(1, 1, 2 ** 31 - 1) > 0
