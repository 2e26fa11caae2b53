"""The 8-bit cache and the attention over it at the ends of the value range."""
import pytest
import torch

from serving_ref import RefCache

pytestmark = pytest.mark.gpu
E4, I8 = torch.float8_e4m3fn, torch.int8
BF16 = torch.bfloat16


def _dev_i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("T", [1, 3, 20])
@pytest.mark.parametrize("small,large", [(1e-30, 1e25), (1e-28, 1e38), (1e-20, 1e20), (1e-30, 1e15)])
def test_append_grid_grows_by_any_factor(T, small, large, dtype):
    """A block that holds tiny rows takes huge ones: on the new grid the older rows are what their codes round to there (nothing, mostly), by whatever
    power of two the grid grew -- factors below the smallest fp32 number among them."""
    from neko_amd import ops
    S, H, cap, hd, block, n0 = 2, 3, 64, 32, 32, 7
    g = torch.Generator().manual_seed(T)
    x = torch.randn(S, n0, 2, H, hd, generator=g).mul(small).to(BF16)
    y = torch.randn(S, T, 2, H, hd, generator=g).mul(large).to(BF16)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    ref = RefCache(S, H, cap, hd, dtype, block)
    for rows, pos in ((x, 0), (y, n0)):
        d = rows.cuda()
        ops.kv8_append(cache, d[:, :, 0], d[:, :, 1], _dev_i([pos] * S))
        ref.append(rows[:, :, 0], rows[:, :, 1], [pos] * S, [rows.shape[1]] * S)
    k, v = ops.kv8_read(cache, _dev_i([n0 + T] * S), cap)
    rk, rv = ref.read([n0 + T] * S, cap)
    assert torch.equal(k.cpu().double(), rk) and torch.equal(v.cpu().double(), rv)


# every kernel: 16 and 32 rows a wave, 128 and 256 rows through LDS, with one split of the keys and several
@pytest.mark.parametrize("hd,S,H,G,T,cap,max_len", [(32, 1, 2, 1, 1, 192, 0), (64, 1, 2, 1, 1, 4096, 0), (64, 2, 2, 4, 6, 4096, 0), (32, 16, 16, 1, 100, 320, 0), (64, 8, 8, 1, 130, 1024, 0),
                                                    (128, 8, 8, 1, 20, 1024, 0), (128, 8, 8, 1, 130, 1024, 0), (128, 2, 4, 1, 520, 1024, 0), (128, 1, 1, 1, 300, 1024, 0)])
@pytest.mark.parametrize("kind", ["all", "some", "rising"])
@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
def test_attn_values_up_to_the_largest(hd, S, H, G, T, cap, max_len, kind, dtype):
    """Visible values up to the largest the cache keeps (what an infinity is stored as): every output is a mean of them and finite.  all: nothing else;
    some: a few positions beside ordinary ones; rising: scores that climb by 2^44 along the keys, the large values at the front (their probabilities
    shrink as the reference moves) or at the back."""
    from neko_amd import ops
    from test_kv8_gpu import _attention_by_heads
    g = torch.Generator().manual_seed(hd + T)
    u = torch.randn(S, 1, H, hd, generator=g).sign()
    k = 0.1 * torch.randn(S, cap, H, hd, generator=g)
    if kind == "rising":                            # q . k hd^-1/2 from -15 to 15 nats
        k = k + torch.linspace(-15.0, 15.0, cap).view(1, cap, 1, 1) * u / hd ** 0.5
    q = (u.repeat_interleave(G, 2) + 0.02 * torch.randn(S, T, H * G, hd, generator=g)).to(BF16)
    v = torch.randn(S, cap, H, hd, generator=g)
    if kind == "all":
        v = v * 3e38                                # infinities among them
    else:
        at = torch.zeros(cap, dtype=torch.bool)
        at[3::97] = True
        at[-1] = True
        v = torch.where(at.view(1, cap, 1, 1), v.sign() * float("inf"), v)
    v = v.to(BF16)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=16 if hd == 128 else 64)
    ops.kv8_append(cache, k.to(BF16).cuda(), v.cuda(), _dev_i([0] * S))
    pos = [cap - T] * S
    got = ops.attn_kv8(cache, q.cuda(), _dev_i(pos), max_len=max_len).cpu().double()
    kk, vv = (t.cpu().double().transpose(1, 2) for t in ops.kv8_read(cache, _dev_i([cap]* S), cap))
    assert bool(torch.isfinite(vv).all()) and float(vv.abs().max()) == 1.75 * 2.0 ** 127
    want, absv, big = _attention_by_heads(q, kk, vv, pos, [T] * S, [0] * S, 0, 0, hd ** -0.5, torch.zeros(S, T, H * G, hd))
    assert bool(torch.isfinite(got).all())
    # as for ordinary values (output rounding, probabilities of 8 or 16 bits, the score's and the exponent's roundings, the sums', the exponential's)
    p_round = 2.0 ** -8 if T * G > 64 else 2.0 ** -16
    tol = 2.0 ** -8 * want.abs() + (p_round + (2 * hd + 8) * 2.0 ** -23 * big + cap * 2.0 ** -23 + 2.0 ** -21) * absv
    err = (got - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
